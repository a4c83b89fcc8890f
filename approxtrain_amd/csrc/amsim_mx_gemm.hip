// Products of MXFP4 operands (amsim_mx.h) on the matrix cores: out[m][n] = act(sum_k a[m][k] b[n][k] + bias[n]).
//
// A 16x16x128 instruction takes 16 bytes of codes and one scale from each lane: a lane's operand is one block of
// 32 values, which is what the storage hands out.  The product of two elements is exact, and so are the sums
// within an instruction but for bits far below the largest term; steps add up in 32 bits.  The operands are
// swapped in the instruction (b's rows are its rows) so that a lane ends up with four neighbouring columns.
//
// Times in these comments compare one thing with another, launches in a row on one device; devices and neighbouring
// kernels move them by some percent (4096^3 in 16 bits 37 to 40 us).
#include "amsim_mx.h"

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

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
    unsigned tiles_m, tiles_n;  // (below 2^24 together)
    int splits;
    int around;              // large results go past the last-level cache
    float *partial;          // [splits][m][n] where the reduction is split, else null
};
// One or two products of a launch: a training step's backward pass has two that do not wait for each other.
struct GemmJobs {
    GemmArgs job[2];
    unsigned blocks;         // of the first
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
__device__ __forceinline__ void finish4(const void *bias, int bias_dtype, int act, void *out, int out_dtype, int64_t m, int64_t n, int64_t N, float (&v)[4])
{
    const int count = (int)(N - n < 4 ? N - n : 4);
    const bool vector = N % 4 == 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (bias && i < count) v[i] += load_as_float(bias, bias_dtype, n + i);
        v[i] = activate(v[i], act);
    }
    if (out_dtype == AMSIM_DTYPE_F32) store4((float *)out + m * N + n, v, count, vector);
    else if (out_dtype == AMSIM_DTYPE_BF16) store4((__bf16 *)out + m * N + n, v, count, vector);
    else store4((_Float16 *)out + m * N + n, v, count, vector);
}

template <int SA, int SB> __device__ __forceinline__ v4f mfma(v4i a, v4i b, v4f c, int sa, int sb)
{
    const v8i wa = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, wb = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, wb, c, 4, 4, SA, sa, SB, sb);
}
// fn(integral_constant 0), ... fn(integral_constant N - 1): indices that are part of an instruction
template <typename Fn, int... I> __device__ __forceinline__ void for_each(Fn &&fn, std::integer_sequence<int, I...>)
{
    (fn(std::integral_constant<int, I>{}), ...);
}
template <int N, typename Fn> __device__ __forceinline__ void for_each(Fn &&fn) { for_each(fn, std::make_integer_sequence<int, N>{}); }

// Where tile number `id` of a launch lies.  Workgroups go to the eight dies in turn; each die gets a run of
// neighbouring tiles, eight tiles high, so that its L2 serves a fragment's step to all who read it.
__device__ __forceinline__ void place_tile(unsigned id, unsigned tiles_m, unsigned tiles_n, unsigned &tm, unsigned &tn)
{
    const unsigned tiles = tiles_m * tiles_n, each = tiles / 8, more = tiles % 8, die = id % 8;
    const unsigned t = die * each + min(die, more) + id / 8;
    const unsigned band = 8 * tiles_n, first = t / band * 8, within = t % band, high = min(8u, tiles_m - first);
    tm = first + within % high;
    tn = within / high;
}

// s_waitcnt for vmcnt n outstanding loads, and for all of LDS's answers
#define MX_WAIT_LOADS(n) __builtin_amdgcn_s_waitcnt(((n) & 15) | 7 << 4 | 15 << 8 | ((n) >> 4) << 14)
#define MX_WAIT_LDS() __builtin_amdgcn_s_waitcnt(15 | 7 << 4 | 0 << 8 | 3 << 14)
// the workgroup meets without waiting for anything else; no access to memory moves across it
__device__ __forceinline__ void meet()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
// what a wavefront wrote to LDS is read by its other lanes after this (LDS answers a wavefront in order)
__device__ __forceinline__ void lanes_meet()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
}

// SIZE bytes a lane from memory to LDS, without passing through registers: lane l's bytes go to to + SIZE l.  The
// wavefront's address and the step's offset stay in scalar registers.
template <int SIZE> __device__ __forceinline__ void load_to_lds(const uint8_t *from, int step_offset, uint8_t *to)
{
#ifdef __HIP_DEVICE_COMPILE__  // (the host's compiler does not know the type)
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void *)from, 0, 0xffffffff, 0x00020000);
    const auto lds = (__attribute__((address_space(3))) void *)to;
    if constexpr (SIZE == 16) __builtin_amdgcn_raw_ptr_buffer_load_lds(r, lds, 16, (threadIdx.x & 63) * 16, step_offset, 0, 0);
    else __builtin_amdgcn_raw_ptr_buffer_load_lds(r, lds, 4, (threadIdx.x & 63) * 4, step_offset, 0, 0);
#endif
}

// A wave's results to memory, by way of LDS: a lane's four columns lie in sixteen rows' lines, a row of 16 F columns
// is whole ones.  The rows' padding puts sixteen rows' writes on different banks.  A tile of 256, alone on its CU,
// goes out in parts (16 rows of 32 bits or 32 of 16), so that its first stores are under way early: 4096^3 takes 37.2 us
// so and 37.6 in one part; tiles of 128 and less, which have neighbours to hide behind, in one: 42.7 and 44.1.
template <typename T, int FM, int FN> struct Rows {
    static constexpr int COLUMNS = 16 * FN, STRIDE = COLUMNS * sizeof(T) + 16, AT_ONCE = FM * FN == 32 ? 32 / FN / sizeof(T) : FM;
    static constexpr int BYTES = 16 * AT_ONCE * STRIDE;
};
template <typename T, int FM, int FN>
__device__ __forceinline__ void store_tile(uint8_t *lds, const v4f (&acc)[FM][FN], const float (&bias)[FN][4], int act, T *out, int64_t m0,
                                           int64_t n0, int64_t M, int64_t N, bool around)
{
    using R = Rows<T, FM, FN>;
    const int lane = threadIdx.x & 63, columns = (int)min<int64_t>(R::COLUMNS, N - n0);
    for_each<FM / R::AT_ONCE>([&](auto part) {
        constexpr int first = part.value * R::AT_ONCE;
        MX_WAIT_LDS();  // (what lay there before has been read)
        for_each<R::AT_ONCE * FN>([&](auto at) {
            constexpr int i = at.value / FN, j = at.value % FN;
            T t[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = from_float<T>(activate(acc[first + i][j][e] + bias[j][e], act));
            __builtin_memcpy(__builtin_assume_aligned(lds + (16 * i + lane % 16) * R::STRIDE + (16 * j + lane / 16 * 4) * sizeof(T), 4 * sizeof(T)), t, sizeof(t));
        });
        lanes_meet();
        const int64_t row0 = m0 + 16 * first;
        const int rows = (int)max<int64_t>(0, min<int64_t>(16 * R::AT_ONCE, M - row0));
        T *o = out + row0 * N + n0;
        constexpr int PIECE = 16 / sizeof(T), PIECES = R::COLUMNS / PIECE, DOWN = 64 / PIECES;  // DOWN: rows that a store covers
        const int c = lane % PIECES * PIECE;
        const uint8_t *from = lds + lane / PIECES * R::STRIDE + c * sizeof(T);
        T *to = o + lane / PIECES * N + c;
        // (rows may start on any element: the hardware takes such pieces too)
        auto pieces = [&](auto past) {
#pragma unroll 8
            for (int r = lane / PIECES; r < 16 * R::AT_ONCE; r += DOWN, from += DOWN * R::STRIDE, to += DOWN * N) {
                const v4i v = *(const v4i *)from;
                if (r >= rows) continue;
                if constexpr (past.value) __builtin_nontemporal_store(v, (v4i_anywhere *)to);
                else store16(to, v);
            }
        };
        if (c + PIECE <= columns) {
            if (around) pieces(std::true_type{});
            else pieces(std::false_type{});
        } else if (c < columns) {
            for (int r = lane / PIECES; r < rows; r += DOWN, from += DOWN * R::STRIDE, to += DOWN * N)
                for (int i = 0; i < columns - c; ++i) to[i] = ((const T *)from)[i];
        }
        lanes_meet();
    });
}

// A workgroup of WM x WN waves, FM x FN fragments each: a tile of 16 FM WM rows and 16 FN WN columns.  Steps of 128 along the
// reduction go from memory to one of STAGES places in LDS without passing through registers (the storage is
// what a wavefront's 16-byte loads deliver, lane by lane), and a step's fragments are read into
// registers while the step before is multiplied.
template <int FM, int FN, int WM, int WN, int STAGES> struct Gemm {
    static constexpr int WAVES = WM * WN, AM = FM * WM, BN = FN * WN;                // fragments of a tile's sides
    static constexpr int GM = AM >= 4 ? AM / 4 : 1, GN = BN >= 4 ? BN / 4 : 1;       // ... and their scale groups
    static constexpr int A = 0, B = AM * 1024, S = B + BN * 1024, BYTES = S + (GM + GN) * 256;
    static constexpr int FROM_A = AM / WAVES, CODES = (AM + BN) / WAVES, SCALES = (GM + GN + WAVES - 1) / WAVES;  // loads of a wave for a step
    static constexpr int LOADS = CODES + SCALES;
    static constexpr int SM = FM >= 4 ? FM / 4 : 1, SN = FN >= 4 ? FN / 4 : 1;       // dwords of four fragments' scales
    static constexpr int READS = FM + FN + (SM + 1) / 2 + (SN + 1) / 2;              // of LDS (two dwords in one)
    struct Registers {
        v4i a[FM], b[FN];
        int sa[SM], sb[SN];
    };
};

template <int FM, int FN, int WM, int WN, int STAGES, int RESIDENT>
__global__ __launch_bounds__(64 * WM * WN, RESIDENT) void gemm_kernel(GemmJobs jobs)
{
    using K = Gemm<FM, FN, WM, WN, STAGES>;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[STAGES * K::BYTES];
    static_assert(K::WAVES * Rows<float, FM, FN>::BYTES <= STAGES * K::BYTES && K::WAVES * Rows<__bf16, FM, FN>::BYTES <= STAGES * K::BYTES, "");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
    const bool other = blockIdx.x >= jobs.blocks;
    const GemmArgs g = jobs.job[other];
    const unsigned id = blockIdx.x - (other ? jobs.blocks : 0), tiles = g.tiles_m * g.tiles_n, split = g.splits > 1 ? id / tiles : 0;
    unsigned tm, tn;
    place_tile(id - split * tiles, g.tiles_m, g.tiles_n, tm, tn);
    const int64_t beg = split * g.steps_per_split, end = min(beg + g.steps_per_split, g.steps);
    const int count = (int)(end - beg);

    // what this wave fetches: fragments of either operand, and 64 rows' scales (where there are fewer groups than waves'
    // loads, some twice)
    const uint8_t *fetch[K::CODES], *fetch_scales[K::SCALES];
    int to[K::CODES], to_scales[K::SCALES];
#pragma unroll
    for (int i = 0; i < K::CODES; ++i) {
        const bool of_a = i < K::FROM_A;
        const int f = of_a ? K::FROM_A * wave + i : (K::CODES - K::FROM_A) * wave + i - K::FROM_A;
        const Operand &o = of_a ? g.a : g.b;
        const int64_t at = min<int64_t>((of_a ? tm * K::AM : tn * K::BN) + f, o.fragments - 1);
        fetch[i] = o.codes + (at * g.steps + beg) * 1024;
        to[i] = (of_a ? K::A : K::B) + f * 1024;
    }
#pragma unroll
    for (int i = 0; i < K::SCALES; ++i) {
        const int group = (wave + K::WAVES * i) % (K::GM + K::GN);
        const bool of_a = group < K::GM;
        const Operand &o = of_a ? g.a : g.b;
        const int64_t at = min<int64_t>(of_a ? tm * K::AM / 4 + group : tn * K::BN / 4 + group - K::GM, o.groups - 1);
        fetch_scales[i] = o.scales + (at * g.steps + beg) * 256;
        to_scales[i] = K::S + group * 256;
    }
    auto fetch_step = [&](int s) {
        uint8_t *stage = lds + s % STAGES * K::BYTES;
        const int at = min(s, count - 1);
#pragma unroll
        for (int i = 0; i < K::CODES; ++i) load_to_lds<16>(fetch[i], at * 1024, stage + to[i]);
#pragma unroll
        for (int i = 0; i < K::SCALES; ++i) load_to_lds<4>(fetch_scales[i], at * 256, stage + to_scales[i]);
    };
    auto read_step = [&](int s, typename K::Registers &r) {
        const uint8_t *stage = lds + s % STAGES * K::BYTES;
#pragma unroll
        for (int i = 0; i < FM; ++i) r.a[i] = *(const v4i *)(stage + K::A + (wm * FM + i) * 1024 + lane * 16);
#pragma unroll
        for (int i = 0; i < FN; ++i) r.b[i] = *(const v4i *)(stage + K::B + (wn * FN + i) * 1024 + lane * 16);
#pragma unroll
        for (int i = 0; i < K::SM; ++i) {
            r.sa[i] = *(const int *)(stage + K::S + (FM >= 4 ? wm * K::SM + i : 0) * 256 + lane * 4);
            if (FM == 2) r.sa[i] >>= 16 * wm;
        }
#pragma unroll
        for (int i = 0; i < K::SN; ++i) {
            r.sb[i] = *(const int *)(stage + K::S + (K::GM + (FN >= 4 ? wn * K::SN + i : 0)) * 256 + lane * 4);
            if (FN == 2) r.sb[i] >>= 16 * wn;
        }
    };
    v4f acc[FM][FN] = {};
    auto multiply = [&](const typename K::Registers &r) {
        for_each<FM * FN>([&](auto at) {
            constexpr int i = at.value / FN, j = at.value % FN;
            acc[i][j] = mfma<j % 4, i % 4>(r.b[j], r.a[i], acc[i][j], r.sb[j / 4], r.sa[i / 4]);
        });
    };
    // One step: everyone has read step s and its successor's loads are in LDS; loads of step s + STAGES take the
    // place of step s; fragments of s + 1 are read while those of s are multiplied.  (Without branches, so that the
    // multiplications stay where they are: behind the last step it is loaded again, and not used.)
    auto step = [&](int s, const typename K::Registers &now, typename K::Registers &next) {
        MX_WAIT_LDS();
        MX_WAIT_LOADS((STAGES - 2) * K::LOADS);
        meet();
        read_step(s + 1, next);
        fetch_step(s + STAGES);
        multiply(now);
        // a read of LDS behind a multiplication, then a load behind every fourth (few fragments: second)
        for_each<K::READS>([](auto) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        });
        for_each<K::LOADS>([](auto) {
            __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, FM * FN == 64 ? 4 : 2, 0);
        });
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int s = 0; s < STAGES; ++s) fetch_step(s);
    MX_WAIT_LOADS((STAGES - 1) * K::LOADS);
    meet();
    typename K::Registers even, odd;
    read_step(0, even);
    int s = count & 1;
    if (s) {
        step(0, even, odd);
        even = odd;
    }
    for (; s < count; s += 2) {
        step(s, even, odd);
        step(s + 1, odd, even);
    }
    MX_WAIT_LDS();
    MX_WAIT_LOADS(0);
    meet();  // (LDS is free)
    const int64_t m0 = (int64_t)(tm * WM + wm) * FM * 16, n0 = (int64_t)(tn * WN + wn) * FN * 16;
    if (m0 >= g.a.rows || n0 >= g.b.rows) return;
    const bool whole = !g.partial;
    float bias[FN][4];
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t n = n0 + 16 * j + lane / 16 * 4 + e;
            bias[j][e] = whole && g.bias && n < g.b.rows ? load_as_float(g.bias, g.bias_dtype, n) : 0.0f;
        }
    auto store = [&](auto zero, auto *out) {
        using T = decltype(zero);
        store_tile<T, FM, FN>(lds + wave * Rows<T, FM, FN>::BYTES, acc, bias, whole ? g.act : AMSIM_ACT_NONE, out, m0, n0, g.a.rows, g.b.rows,
                              whole && g.around);
    };
    if (!whole || g.out_dtype == AMSIM_DTYPE_F32) store(0.0f, whole ? (float *)g.out : g.partial + split * g.a.rows * g.b.rows);
    else if (g.out_dtype == AMSIM_DTYPE_BF16) store((__bf16)0.0f, (__bf16 *)g.out);
    else store((_Float16)0.0f, (_Float16 *)g.out);
}

// Few rows: bound by the reading of b, and for one layer of one token by latency alone.  A workgroup takes 16
// of b's rows and the whole reduction, its waves every n-th step each; their sums meet in LDS and are added in order.
struct FewArgs {
    Operand b, a;            // a: of few_kernel
    const void *x;           // of raw_kernel: [rows][k], rows row_stride elements apart
    int64_t row_stride, rows, k, steps;
    const void *bias;
    int bias_dtype, act, out_dtype;
    void *out;
};
constexpr int AHEAD = 4;     // steps of b that a wave has under way at once

// (behind the last step it is loaded again, and not used)
struct FewSteps {
    v4i codes[AHEAD];
    int scales[AHEAD];
    __device__ __forceinline__ void load(const FewArgs &g, int64_t f, int64_t s, int waves)
    {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) {
            const int64_t t = min<int64_t>(s + h * waves, g.steps - 1);
            codes[h] = *(const v4i *)(g.b.codes + ((f * g.steps + t) * 64 + lane) * 16);
            scales[h] = g.b.scales[((f / 4 * g.steps + t) * 64 + lane) * 4 + f % 4];
        }
    }
};

// the fragments' sums over the waves and their results, a fragment to a wave
template <int FA> __device__ __forceinline__ void finish_few(const FewArgs &g, int64_t f, v4f *sums, const v4f (&acc)[FA])
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
#pragma unroll
    for (int i = 0; i < FA; ++i) sums[(wave * FA + i) * 64 + lane] = acc[i];
    __syncthreads();
    for (int i = wave; i < FA; i += waves) {
        v4f z = sums[i * 64 + lane];
        for (int w = 1; w < waves; ++w) z += sums[(w * FA + i) * 64 + lane];
        const int64_t m = 16 * i + lane % 16, n = f * 16 + lane / 16 * 4, N = g.b.rows;
        if (m >= g.rows || n >= N) continue;
        float v[4] = {z[0], z[1], z[2], z[3]};
        finish4(g.bias, g.bias_dtype, g.act, g.out, g.out_dtype, m, n, N, v);
    }
}

// FA fragments of converted rows.
template <int FA>
__global__ __launch_bounds__(1024) void few_kernel(FewArgs g)
{
    __shared__ v4f sums[16 * FA * 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    v4f acc[FA] = {};
    for (int64_t s = wave; s < g.steps; s += AHEAD * waves) {
        FewSteps b;
        b.load(g, blockIdx.x, s, waves);
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) {
            const int64_t t = s + h * waves;
            if (t >= g.steps) break;
            v4i a[FA];
#pragma unroll
            for (int i = 0; i < FA; ++i) a[i] = *(const v4i *)(g.a.codes + ((min<int64_t>(i, g.a.fragments - 1) * g.steps + t) * 64 + lane) * 16);
            const int ca = *(const int *)(g.a.scales + (t * 64 + lane) * 4);
            for_each<FA>([&](auto i) { acc[i.value] = mfma<0, i.value>(b.codes[h], a[i.value], acc[i.value], b.scales[h], ca); });
        }
    }
    finish_few(g, blockIdx.x, sums, acc);
}

// FA fragments of rows as they come: every workgroup converts them for itself, into LDS, four lanes to a block, while
// its first loads of b are under way.  That saves a launch, and for a token's layer half the time.
constexpr int64_t RAW_VALUES = 32768;  // rows x length (in whole steps) that it converts
template <typename X, int FA>
__global__ __launch_bounds__(1024) void raw_kernel(FewArgs g)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t converted[];  // codes [block][row][16 bytes], scales [block][row]; then the sums
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int rows = (int)g.rows, apart = rows | 1, blocks = (int)g.steps * 4;  // (an odd distance: a row's blocks lie in different banks)
    uint8_t *scales = converted + blocks * apart * 16;
    FewSteps b;
    b.load(g, blockIdx.x, wave, waves);
    const int eighths = blocks * 4, down = blockDim.x / eighths, across = blockDim.x % eighths;
    int r = threadIdx.x / eighths, e8 = threadIdx.x % eighths;
    while (r < rows) {  // (a block's four lanes stay together)
        constexpr int BATCH = 2;
        X v[BATCH][8] = {};
        int row[BATCH], eighth[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
            row[j] = r, eighth[j] = e8;
            r += down, e8 += across;
            if (e8 >= eighths) e8 -= eighths, ++r;
            if (row[j] >= rows) continue;
            const X *p = (const X *)g.x + row[j] * g.row_stride + eighth[j] * 8;
            if (eighth[j] * 8 + 8 <= g.k) {
                v4i piece[sizeof(v[j]) / 16];
#pragma unroll
                for (int e = 0; e < (int)(sizeof(v[j]) / 16); ++e) piece[e] = load16((const char *)p + 16 * e);
                __builtin_memcpy(v[j], piece, sizeof(v[j]));
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (eighth[j] * 8 + e < g.k) v[j][e] = p[e];
            }
        }
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
            if (row[j] >= rows) break;
            uint32_t largest = mx_exponent_field(v[j]);
            largest = max(largest, (uint32_t)__shfl_xor((int)largest, 1, 64));
            largest = max(largest, (uint32_t)__shfl_xor((int)largest, 2, 64));
            const uint32_t code = mx_scale_code(largest);
            const int at = eighth[j] / 4 * apart + row[j];
            *(uint32_t *)(converted + at * 16 + eighth[j] % 4 * 4) = mx_encode8(v[j], code);
            if (eighth[j] % 4 == 0) scales[at] = (uint8_t)code;
        }
    }
    __syncthreads();
    int row[FA];
#pragma unroll
    for (int i = 0; i < FA; ++i) row[i] = min(16 * i + lane % 16, rows - 1);  // (results of rows that do not exist are not stored)
    v4f acc[FA] = {};
    for (int64_t s = wave; s < g.steps; s += AHEAD * waves) {
        if (s != wave) b.load(g, blockIdx.x, s, waves);
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) {
            const int t = (int)s + h * waves;
            if (t >= g.steps) break;
#pragma unroll
            for (int i = 0; i < FA; ++i) {
                const int at = (4 * t + lane / 16) * apart + row[i];
                acc[i] = mfma<0, 0>(b.codes[h], *(const v4i *)(converted + at * 16), acc[i], b.scales[h], scales[at]);
            }
        }
    }
    __syncthreads();  // (the sums take the place of what was converted)
    finish_few(g, blockIdx.x, (v4f *)converted, acc);
}

// What is left behind the products: partial sums of split reductions, added in the order of the splits, and a bias
// gradient's from the sums of every 32 rows, 16 columns and 64 runs of rows to a workgroup, the runs joined in pairs.
constexpr int FINISH_WG = 1024, MOST_SPLITS = 16;
struct FinishArgs {
    GemmJobs products;
    unsigned blocks[2];      // of either product's sums
    const float *sums;       // [parts][columns]
    int64_t parts, columns;
    void *out;
    int out_dtype;
};
__global__ __launch_bounds__(FINISH_WG) void finish_kernel(FinishArgs f)
{
    constexpr int RUNS = FINISH_WG / 16;
    __shared__ float run[RUNS][16];
    unsigned id = blockIdx.x;
    if (id < f.blocks[0] + f.blocks[1]) {
        const bool other = id >= f.blocks[0];
        if (other) id -= f.blocks[0];
        const GemmArgs &g = f.products.job[other];
        const int64_t N = g.b.rows, quads = ceil_div64(N, 4), at = (int64_t)id * FINISH_WG + threadIdx.x;
        if (at >= g.a.rows * quads) return;
        const int64_t m = at / quads, n = at % quads * 4;
        const int count = (int)(N - n < 4 ? N - n : 4);
        const float *p = g.partial + m * N + n;
        const int64_t apart = g.a.rows * N;
        v4f part[MOST_SPLITS];  // (all under way at once: one after the other they take a microsecond each)
#pragma unroll
        for (int s = 0; s < MOST_SPLITS; ++s) {
            part[s] = v4f{0, 0, 0, 0};
            if (s >= g.splits) continue;
            if (count == 4) {
                part[s] = __builtin_bit_cast(v4f, load16(p + s * apart));
            } else {
#pragma unroll
                for (int i = 0; i < 3; ++i)
                    if (i < count) part[s][i] = p[s * apart + i];
            }
        }
        float v[4] = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < MOST_SPLITS; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += part[s][i];
        finish4(g.bias, g.bias_dtype, g.act, g.out, g.out_dtype, m, n, N, v);
        return;
    }
    id -= f.blocks[0] + f.blocks[1];
    const int c = threadIdx.x & 15, w = threadIdx.x >> 4;
    const int64_t col = (int64_t)id * 16 + c, each = ceil_div64(f.parts, RUNS), end = min(f.parts, each * (w + 1));
    float s = 0.0f;
    if (col < f.columns) {
#pragma unroll 8
        for (int64_t p = each * w; p < end; ++p) s += f.sums[p * f.columns + col];
    }
    run[w][c] = s;
    for (int half = RUNS / 2; half; half /= 2) {
        __syncthreads();
        if (w < half) run[w][c] += run[w + half][c];
    }
    if (w != 0 || col >= f.columns) return;
    s = run[0][c];
    if (f.out_dtype == AMSIM_DTYPE_F32) ((float *)f.out)[col] = s;
    else if (f.out_dtype == AMSIM_DTYPE_BF16) ((__bf16 *)f.out)[col] = (__bf16)s;
    else ((_Float16 *)f.out)[col] = (_Float16)s;
}

struct Tile {
    int rows, cols, slots;  // slots: tiles that the card holds at once
    // microseconds, as measured on products of 128 to 16384 a side: of a launch; of a step where a tile has a CU for itself,
    // and where all slots are taken; of storing a tile (between results of 16 bits and of 32: workspaces are asked for
    // before the type is known)
    double base, alone, full, store;
};
// Tiles of 256 fetch least for an operation and have their CU for themselves, with eight waves (four with twice the
// fragments: 39.8 us for 4096^3, 37.1 with eight): what they store, nobody multiplies beside.  256 x 128 share it by two (512
// tiles of 32 steps: 38.7 us, 37.1 as 256 of 256, 42.2 as 1024 of 128; of 128 steps 124, 112 and 136; 2048 tiles of 16 steps
// 84, 89, 92).  Tiles of 128 and 64 fetch two and four times the bytes, and are for few results (256 tiles of 128, 16
// steps: 10.0 us, 13.9 in 256 x 128; 410 of 64, 21 steps: 7.7, 10.1 in 128).
constexpr Tile TILES[] = {{256, 256, 256, 2.2, 0.55, 0.785, 10.8},  // (stored by a round at once)
                          {256, 128, 512, 6.5, 0.5, 0.85, 0.0124}, {128, 128, 512, 5, 0.2, 0.46, 0.01}, {64, 64, 1024, 4, 0.1, 0.4, 0.003}};

struct Extents {
    int64_t m, n, k;
};
struct Plan {
    int tile;  // of TILES
    struct {
        int64_t tiles_m, tiles_n, splits, steps_per_split;
    } of[2];
};

// What a launch of `tiles` tiles takes whose steps add up to `work` and are at most `longest`: rounds of all slots, and a
// last one in which a CU has one tile or a few.
double microseconds(int tile, double tiles, double work, double longest)
{
    const Tile &t = TILES[tile];
    const double mean = work / tiles, rounds = std::floor(tiles / t.slots), rest = tiles - rounds * t.slots;
    double last = rest > 0 ? std::max(t.alone, t.full * rest / t.slots) : 0;
    if (tile == 1 && rest > 256) last = 0.8;
    const double steps = std::max(rounds * t.full * mean + last * mean, t.alone * longest);
    if (tile == 0) return t.base + std::ceil(tiles / t.slots) * (t.store + 1.5) - 1.5 + steps;
    return t.base + steps + t.store * tiles;
}

// The tile of one or two products and the splits of their reductions that take least time.  A split reduction takes a
// second launch, 3 us, and its sums go to memory and back.
Plan make_plan(const Extents *e, int count)
{
    Plan best{-1, {}};
    double least = 0;
    for (int i = 0; i < 4; ++i) {
        Plan p{i, {}};
        double tiles = 0, work = 0, longest = 0, more = 0;
        for (int j = 0; j < count; ++j) {
            const int64_t steps = mx_steps(e[j].k), tiles_m = ceil_div64(e[j].m, TILES[i].rows), tiles_n = ceil_div64(e[j].n, TILES[i].cols);
            const double area = (double)tiles_m * (double)tiles_n;
            double quickest = 0, its_more = 0;
            for (int64_t s = 1; s <= MOST_SPLITS && (s == 1 || 2 * s <= steps); s *= 2) {
                const int64_t each = ceil_div64(steps, s), splits = ceil_div64(steps, each);
                const double extra = splits > 1 ? 3 + (double)splits * (double)e[j].m * (double)e[j].n * 8 / 4e6 : 0;
                const double us = microseconds(i, area * splits, area * splits * each, each) + extra;
                if (s > 1 && us >= quickest) continue;
                quickest = us;
                its_more = extra;
                p.of[j] = {tiles_m, tiles_n, splits, each};
            }
            const double all = area * p.of[j].splits;
            tiles += all;
            work += all * p.of[j].steps_per_split;
            longest = std::max(longest, (double)p.of[j].steps_per_split);
            more += its_more;
        }
        const double us = microseconds(i, tiles, work, longest) + more;
        if (best.tile < 0 || us < least) {
            least = us;
            best = p;
        }
    }
    return best;
}

// The same, looked up where the thread has asked for it before: a training step asks seven times, a microsecond each.
Plan plan(const Extents *e, int count)
{
    struct Known {
        Extents e[2];
        Plan p;
    };
    static thread_local Known known[64] = {};
    const Extents none{}, &f = count > 1 ? e[1] : none;
    const uint64_t hash = ((uint64_t)e[0].m * 3 + (uint64_t)e[0].n * 5 + (uint64_t)e[0].k * 7 + (uint64_t)f.k * 11) * 0x9e3779b97f4a7c15ull;
    Known &at = known[hash >> 58];
    auto same = [](const Extents &x, const Extents &y) { return x.m == y.m && x.n == y.n && x.k == y.k; };
    if (!same(at.e[0], e[0]) || !same(at.e[1], f)) at = Known{{e[0], f}, make_plan(e, count)};
    return at.p;
}

// Whether few_kernel serves, by rows and length alone: a reduction beyond 32768 needs more than one workgroup's waves.  us of
// the product by itself, few_kernel / tiles, of 16, 32 and 64 rows:
//   length    10 wide                          512 wide                         8192 wide
//     2048    3.3/5.2   3.7/5.5   4.6/5.6      3.5/5.2   3.9/5.3   4.8/5.3       4.7/5.3   5.6/5.5   7.7/5.6
//     8192    4.1/7.7   4.9/7.9   6.4/8.1      4.5/8.8   5.4/8.1   6.7/8.4       9.4/12.7  10.9/12.8 15.5/12.9
//    16384    5.6/8.3   6.8/8.6   9.2/8.9      6.0/9.2   7.2/9.7   9.5/10.0     15.0/17.0  16.5/17.5 27.6/18.4
//    32768    8.7/9.2  10.7/9.5  14.7/10.2     9.1/10.5 11.2/10.7 15.0/11.3     27.3/27.6  29.1/27.8 50.4/29.3
// Of 240 such products (1, 16, 17, 32 and 64 rows, 10 to 8192 wide, lengths of 128 to 32768) it takes 1.03 times the quicker's
// time on average.  Tiles are quicker by a tenth or more for 64 rows of a length of 128, 64 rows that are 8192 wide or of
// 16384 and more, and at 32768 from 17 rows on where few are wide.
bool few(int64_t m, int64_t k) { return m <= 64 && mx_steps(k) <= 256; }

size_t partial_bytes(const Extents &e, int64_t splits) { return splits > 1 ? ((size_t)splits * e.m * e.n * 4 + 255) / 256 * 256 : 0; }

// the products of a list that go in tiles, and the others
int tiled(const Extents *e, int count, Extents *out, int *which)
{
    int n = 0;
    for (int j = 0; j < count; ++j)
        if (!few(e[j].m, e[j].k)) out[n] = e[j], which[n++] = j;
    return n;
}

size_t products_workspace(const Extents *e, int count)
{
    Extents t[2];
    int which[2];
    const int n = tiled(e, count, t, which);
    if (n == 0) return 0;
    const Plan p = plan(t, n);
    size_t bytes = 0;
    for (int j = 0; j < n; ++j) bytes += partial_bytes(t[j], p.of[j].splits);
    return bytes;
}
size_t product_workspace(int64_t m, int64_t n, int64_t k)
{
    const Extents e{m, n, k};
    return products_workspace(&e, 1);
}

// A wave for every step, and for 128 of the pieces of 8 values that are to be converted first (64 rows of 128: 16 waves
// 4.7 us, one 8.7).
int few_waves(const FewArgs &g, int64_t pieces)
{
    int waves = 1;
    while (waves < 16 && (waves < g.steps || 128 * waves < pieces)) waves *= 2;
    return waves;
}
int launch_few(void (*kernel)(FewArgs), const FewArgs &g, int waves, int64_t lds, hipStream_t stream)
{
    if (g.b.fragments >= (1ll << 22)) return fail(AMSIM_ERR_UNSUPPORTED, "mxfp4: more tiles than one launch takes");
    kernel<<<(unsigned)g.b.fragments, 64 * waves, lds, stream>>>(g);
    AMSIM_HIP_CHECK(hipGetLastError());
    return AMSIM_OK;
}
template <typename X> int launch_raw(const FewArgs &g, hipStream_t stream)
{
    const int fragments = g.rows <= 16 ? 1 : g.rows <= 32 ? 2 : 4, waves = few_waves(g, g.rows * g.steps * 16);
    const int64_t lds = std::max<int64_t>(g.steps * 4 * (g.rows | 1) * 17, waves * fragments * 1024);
    return launch_few(fragments == 1 ? raw_kernel<X, 1> : fragments == 2 ? raw_kernel<X, 2> : raw_kernel<X, 4>, g, waves, lds, stream);
}

struct Product {
    Operand a, b;
    int64_t k;
    const void *bias;
    int bias_dtype, act;
    void *out;
    int out_dtype;
};

// One or two products, and the sums of `parts` rows of `columns` partial ones where `sums` is not null.
int products(const Product *list, int count, const float *sums, int64_t parts, int64_t columns, void *out, int out_dtype, void *workspace,
             hipStream_t stream)
{
    Extents e[2], t[2];
    int which[2];
    for (int j = 0; j < count; ++j) e[j] = {list[j].a.rows, list[j].b.rows, list[j].k};
    const int n = tiled(e, count, t, which);
    for (int j = 0; j < count; ++j) {
        const Product &q = list[j];
        if (!few(e[j].m, e[j].k)) continue;
        const FewArgs f{q.b, q.a, nullptr, 0, q.a.rows, q.k, mx_steps(q.k), q.bias, q.bias_dtype, q.act, q.out_dtype, q.out};
        if (int rc = launch_few(q.a.rows <= 16 ? few_kernel<1> : q.a.rows <= 32 ? few_kernel<2> : few_kernel<4>, f, few_waves(f, 0), 0, stream)) return rc;
    }
    FinishArgs f{};
    if (n) {
        Plan p = plan(t, n);
        if (n == 2 && p.of[1].steps_per_split > p.of[0].steps_per_split)  // the tiles that take longest go first
            std::swap(t[0], t[1]), std::swap(which[0], which[1]), std::swap(p.of[0], p.of[1]);
        GemmJobs &jobs = f.products;
        int64_t blocks = 0;
        char *partial = (char *)workspace;
        for (int j = 0; j < n; ++j) {
            const Product &q = list[which[j]];
            const auto &o = p.of[j];
            jobs.job[j] = GemmArgs{q.a, q.b, mx_steps(q.k), o.steps_per_split, q.bias, q.bias_dtype, q.act, q.out_dtype, q.out, (unsigned)o.tiles_m,
                                   (unsigned)o.tiles_n, (int)o.splits, mx_goes_around((double)t[j].m * (double)t[j].n * element_bytes(q.out_dtype)),
                                   o.splits > 1 ? (float *)partial : nullptr};
            partial += partial_bytes(t[j], o.splits);
            if (j == 0) jobs.blocks = (unsigned)std::min<int64_t>(o.tiles_m * o.tiles_n * o.splits, 1 << 30);
            blocks += o.tiles_m * o.tiles_n * o.splits;
            if (o.splits > 1) f.blocks[j] = (unsigned)ceil_div64(t[j].m * ceil_div64(t[j].n, 4), FINISH_WG);
            // (steps are counted in 32-bit offsets of 1 KB)
            if (blocks >= (1ll << 24) || o.steps_per_split >= (1ll << 21)) return fail(AMSIM_ERR_UNSUPPORTED, "mxfp4: more tiles or steps than one launch takes");
        }
        switch (p.tile) {
        case 0: gemm_kernel<4, 8, 4, 2, 4, 2><<<(unsigned)blocks, 512, 0, stream>>>(jobs); break;
        case 1: gemm_kernel<8, 4, 2, 2, 3, 2><<<(unsigned)blocks, WG, 0, stream>>>(jobs); break;
        case 2: gemm_kernel<4, 4, 2, 2, 4, 2><<<(unsigned)blocks, WG, 0, stream>>>(jobs); break;
        default: gemm_kernel<2, 2, 2, 2, 4, 4><<<(unsigned)blocks, WG, 0, stream>>>(jobs); break;
        }
        AMSIM_HIP_CHECK(hipGetLastError());
    }
    f.sums = sums, f.parts = parts, f.columns = columns, f.out = out, f.out_dtype = out_dtype;
    const unsigned last = f.blocks[0] + f.blocks[1] + (sums ? (unsigned)ceil_div64(columns, 16) : 0);
    if (last) {
        finish_kernel<<<last, FINISH_WG, 0, stream>>>(f);
        AMSIM_HIP_CHECK(hipGetLastError());
    }
    return AMSIM_OK;
}
int product(const Product &q, void *workspace, hipStream_t stream) { return products(&q, 1, nullptr, 0, 0, nullptr, 0, workspace, stream); }

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

// Whether few rows are converted by every workgroup that multiplies them, not once ahead, by a launch of 3 us (and as
// much again of the host).  Rows x length of 32768 cost a round of 256 workgroups what that launch costs: 8 rows through
// 4096 x 4096 take 7.0 us so, 7.7 converted ahead; 16 rows of 1024 x 4096 5.4 and 6.5, 32 rows 6.8 and 6.5; 24 rows of
// 1200 x 1000 6.8 and 7.4, 32 rows 7.9 and 7.4; 48 rows of 640 x 1024 6.7 and 7.0, 64 rows 7.7 and 7.0.
bool converts_on_the_way(int64_t m, int64_t n, int64_t k)
{
    const int64_t values = m * mx_steps(k) * 128;
    return m <= 64 && values * ceil_div64(n, 4096) <= RAW_VALUES;
}

size_t operand_bytes(int64_t rows, int64_t length) { return (size_t)(mx_code_bytes(rows, length) + mx_scale_bytes(rows, length)); }
size_t sums_bytes(int64_t m, int64_t n) { return ((size_t)ceil_div64(m, 32) * n * 4 + 255) / 256 * 256; }

bool product_fits(int64_t m, int64_t n, int64_t k)
{
    return mx_extents_fit(m, k) && mx_extents_fit(n, k) && mx_extents_fit(m, n) && m && n && k;
}

}  // namespace

}  // namespace amsim

using namespace amsim;

extern "C" {

int amsim_mxfp4_plan(int count, const int64_t *extents, int64_t *info)
{
    if (count < 1 || count > 2 || !extents || !info) return fail(AMSIM_ERR_INVALID, "mxfp4: one or two products are planned");
    Extents e[2], t[2];
    int which[2];
    for (int j = 0; j < count; ++j) {
        e[j] = {extents[3 * j], extents[3 * j + 1], extents[3 * j + 2]};
        if (!product_fits(e[j].m, e[j].n, e[j].k)) return fail(AMSIM_ERR_UNSUPPORTED, "mxfp4: extents out of range");
    }
    info[0] = info[1] = info[2] = info[3] = 0;
    if (const int n = tiled(e, count, t, which)) {
        const Plan p = plan(t, n);
        info[0] = TILES[p.tile].rows, info[1] = TILES[p.tile].cols;
        for (int j = 0; j < n; ++j) info[2 + which[j]] = p.of[j].splits;
    }
    return AMSIM_OK;
}

size_t amsim_mxfp4_matmul_workspace_bytes(int64_t m, int64_t n, int64_t k)
{
    return product_fits(m, n, k) ? product_workspace(m, n, k) : 0;
}

int amsim_mxfp4_matmul(const void *a, const void *b, int64_t m, int64_t n, int64_t k, const void *bias, int bias_dtype, int act,
                       void *out, int out_dtype, void *workspace, size_t workspace_bytes, void *stream)
{
    if (int rc = check_product(m, n, k, bias, bias_dtype, act, out, out_dtype)) return rc;
    if (!a || !b) return fail(AMSIM_ERR_INVALID, "mxfp4: null pointer");
    if (((uintptr_t)a & 15) || ((uintptr_t)b & 15)) return fail(AMSIM_ERR_INVALID, "mxfp4: misaligned pointer");
    if (int rc = check_workspace(workspace, workspace_bytes, product_workspace(m, n, k))) return rc;
    return product({operand(a, m, k), operand(b, n, k), k, bias, bias_dtype, act, out, out_dtype}, workspace, (hipStream_t)stream);
}

size_t amsim_mxfp4_linear_workspace_bytes(int64_t m, int64_t n, int64_t k)
{
    if (!product_fits(m, n, k) || converts_on_the_way(m, n, k)) return 0;
    return operand_bytes(m, k) + product_workspace(m, n, k);
}

int amsim_mxfp4_linear(const void *x, int dtype, int64_t row_stride, const void *w, int64_t m, int64_t n, int64_t k, const void *bias,
                       int bias_dtype, int act, void *out, void *workspace, size_t workspace_bytes, void *stream)
{
    if (int rc = check_product(m, n, k, bias, bias_dtype, act, out, dtype)) return rc;
    if (!x || !w) return fail(AMSIM_ERR_INVALID, "mxfp4: null pointer");
    if (row_stride < k && m > 1) return fail(AMSIM_ERR_INVALID, "mxfp4: rows overlap");
    if (((uintptr_t)x & (element_bytes(dtype) - 1)) || ((uintptr_t)w & 15)) return fail(AMSIM_ERR_INVALID, "mxfp4: misaligned pointer");
    if (int rc = check_workspace(workspace, workspace_bytes, amsim_mxfp4_linear_workspace_bytes(m, n, k))) return rc;
    if (converts_on_the_way(m, n, k)) {
        const FewArgs f{operand(w, n, k), {}, x, row_stride, m, k, mx_steps(k), bias, bias_dtype, act, dtype, out};
        switch (dtype) {
        case AMSIM_DTYPE_F32: return launch_raw<float>(f, (hipStream_t)stream);
        case AMSIM_DTYPE_BF16: return launch_raw<__bf16>(f, (hipStream_t)stream);
        default: return launch_raw<_Float16>(f, (hipStream_t)stream);
        }
    }
    const MxConversion job{x, nullptr, dtype, m, k, row_stride, (uint8_t *)workspace, nullptr, nullptr};
    if (int rc = mx_convert(&job, 1, (hipStream_t)stream)) return rc;
    return product({operand(workspace, m, k), operand(w, n, k), k, bias, bias_dtype, act, out, dtype}, (char *)workspace + operand_bytes(m, k),
                   (hipStream_t)stream);
}

size_t amsim_mxfp4_dense_workspace_bytes(int64_t m, int64_t n, int64_t k)
{
    return product_fits(m, n, k) ? operand_bytes(m, k) + operand_bytes(n, k) + product_workspace(m, n, k) : 0;
}

int amsim_mxfp4_dense(const void *x, int dtype, int64_t row_stride, const void *kernel, int kernel_dtype, int64_t kernel_row_stride,
                      int64_t m, int64_t n, int64_t k, const void *bias, int bias_dtype, int act, void *out, void *x_columns,
                      void *kernel_rows, void *workspace, size_t workspace_bytes, void *stream)
{
    if (int rc = check_product(m, n, k, bias, bias_dtype, act, out, dtype)) return rc;
    if (!known_dtype(kernel_dtype)) return fail(AMSIM_ERR_INVALID, "mxfp4: unknown element type");
    if (!x || !kernel) return fail(AMSIM_ERR_INVALID, "mxfp4: null pointer");
    if ((row_stride < k && m > 1) || (kernel_row_stride < n && k > 1)) return fail(AMSIM_ERR_INVALID, "mxfp4: rows overlap");
    if (((uintptr_t)x & (element_bytes(dtype) - 1)) || ((uintptr_t)kernel & (element_bytes(kernel_dtype) - 1)) || ((uintptr_t)x_columns & 15)
        || ((uintptr_t)kernel_rows & 15))
        return fail(AMSIM_ERR_INVALID, "mxfp4: misaligned pointer");
    if (int rc = check_workspace(workspace, workspace_bytes, amsim_mxfp4_dense_workspace_bytes(m, n, k))) return rc;
    uint8_t *x_rows = (uint8_t *)workspace, *kernel_columns = x_rows + operand_bytes(m, k);
    const MxConversion jobs[2] = {{x, nullptr, dtype, m, k, row_stride, x_rows, (uint8_t *)x_columns, nullptr},
                                  {kernel, nullptr, kernel_dtype, k, n, kernel_row_stride, (uint8_t *)kernel_rows, kernel_columns, nullptr}};
    if (int rc = mx_convert(jobs, 2, (hipStream_t)stream)) return rc;
    return product({operand(x_rows, m, k), operand(kernel_columns, n, k), k, bias, bias_dtype, act, out, dtype}, kernel_columns + operand_bytes(n, k),
                   (hipStream_t)stream);
}

size_t amsim_mxfp4_dense_grad_workspace_bytes(int64_t m, int64_t n, int64_t k)
{
    if (!product_fits(m, n, k)) return 0;
    const Extents e[2] = {{m, k, n}, {k, n, m}};
    // (the products of either gradient alone are planned by themselves)
    return operand_bytes(m, n) + operand_bytes(n, m) + sums_bytes(m, n) + std::max({products_workspace(e, 2), products_workspace(e, 1), products_workspace(e + 1, 1)});
}

int amsim_mxfp4_dense_grad(const void *grad, int dtype, int64_t row_stride, const void *out, const void *x_columns, const void *kernel_rows,
                           int64_t m, int64_t n, int64_t k, void *grad_x, void *grad_kernel, int kernel_dtype, void *grad_bias, int bias_dtype,
                           void *workspace, size_t workspace_bytes, void *stream)
{
    if (!known_dtype(dtype) || (grad_kernel && !known_dtype(kernel_dtype)) || (grad_bias && !known_dtype(bias_dtype)))
        return fail(AMSIM_ERR_INVALID, "mxfp4: unknown element type");
    if (!mx_extents_fit(m, k) || !mx_extents_fit(n, k) || !mx_extents_fit(m, n)) return fail(AMSIM_ERR_UNSUPPORTED, "mxfp4: extents out of range");
    if (m == 0 || n == 0 || k == 0) return fail(AMSIM_ERR_INVALID, "mxfp4: empty product");
    if (row_stride < n && m > 1) return fail(AMSIM_ERR_INVALID, "mxfp4: rows overlap");
    if (grad_bias && ceil_div64(n, 16) >= (1ll << 32) / FINISH_WG) return fail(AMSIM_ERR_UNSUPPORTED, "mxfp4: more columns than one launch sums");
    if (!grad || (grad_x && !kernel_rows) || (grad_kernel && !x_columns)) return fail(AMSIM_ERR_INVALID, "mxfp4: null pointer");
    const uintptr_t element = element_bytes(dtype) - 1;
    if (((uintptr_t)grad & element) || ((uintptr_t)out & element) || ((uintptr_t)x_columns & 15) || ((uintptr_t)kernel_rows & 15)
        || ((uintptr_t)grad_x & 15) || ((uintptr_t)grad_kernel & 15) || (grad_bias && ((uintptr_t)grad_bias & (element_bytes(bias_dtype) - 1))))
        return fail(AMSIM_ERR_INVALID, "mxfp4: misaligned pointer");
    if (int rc = check_workspace(workspace, workspace_bytes, amsim_mxfp4_dense_grad_workspace_bytes(m, n, k))) return rc;
    if (!grad_x && !grad_kernel && !grad_bias) return AMSIM_OK;
    hipStream_t s = (hipStream_t)stream;
    uint8_t *rows = (uint8_t *)workspace, *columns = rows + operand_bytes(m, n);
    float *sums = (float *)(columns + operand_bytes(n, m));
    char *partial = (char *)sums + sums_bytes(m, n);
    const MxConversion job{grad, out, dtype, m, n, row_stride, grad_x ? rows : nullptr, grad_kernel ? columns : nullptr, grad_bias ? sums : nullptr};
    if (int rc = mx_convert(&job, 1, s)) return rc;
    Product list[2];
    int count = 0;
    if (grad_x) list[count++] = {operand(rows, m, n), operand(kernel_rows, k, n), n, nullptr, 0, AMSIM_ACT_NONE, grad_x, dtype};
    if (grad_kernel) list[count++] = {operand(x_columns, k, m), operand(columns, n, m), m, nullptr, 0, AMSIM_ACT_NONE, grad_kernel, kernel_dtype};
    return products(list, count, grad_bias ? sums : nullptr, ceil_div64(m, 32), n, grad_bias, bias_dtype, partial, s);
}

}  // extern "C"
