// Products of 8-bit operands (amsim_i8.h) on the matrix cores:
//   out[m][n] = act(float(sum_k a[m][k] b[n][k]) * sa[m] * sb[n] + bias[n]), the sum exact in 32-bit integers.
//
// A 16x16x64 instruction takes 16 bytes of codes from each lane, which is what the storage hands out.  The operands are
// swapped in the instruction (b's rows are its rows) so that a lane ends up with four neighbouring columns.  A sum
// has at most 131072 terms (127^2 * 131072 < 2^31); longer reductions are split, and the parts are added in 64 bits: a result
// depends on no order, and is rounded to 32 bits once before it is scaled.
#include "amsim_i8.h"
#include "amsim_tiles.h"

namespace amsim {

namespace {

constexpr int WG = 256;

struct Operand {
    const uint8_t *codes;
    const float *scales;  // of its rows, or null: ones
    int64_t rows, fragments;
};
inline Operand operand(const void *codes, const void *scales, int64_t rows) { return Operand{(const uint8_t *)codes, (const float *)scales, rows, ceil_div64(rows, 16)}; }
inline Operand operand(const void *q, int64_t rows, int64_t length) { return operand(q, (const uint8_t *)q + i8_code_bytes(rows, length), rows); }

struct GemmArgs {
    Operand a, b;
    int64_t steps, steps_per_split;
    const void *bias;
    int bias_dtype, act, out_dtype;
    void *out;
    unsigned tiles_m, tiles_n;  // (below 2^24 together)
    int splits;
    int around;              // large results go past the last-level cache
    int *partial;            // [splits][m][n] where the reduction is split, else null
};
struct GemmJobs {
    GemmArgs job[2];
    unsigned blocks;         // of the first
};

// sum * a * b, two roundings, that leaves the range of 32 bits only where the result does.  Within 2^-60 .. 2^60 either product
// does so by itself (a whole number is 0 or from 1 to 2^31); other scales are multiplied as fractions, their powers of two
// applied behind, which moves no rounding: a result does not depend on which way its neighbours go.  A NaN stays one.
__device__ __forceinline__ bool plain_scale(float s) { return s >= 0x1p-60f && s <= 0x1p60f; }
__device__ __forceinline__ float scaled_any(float sum, float a, float b)
{
    const int ea = __builtin_amdgcn_frexp_expf(a), eb = __builtin_amdgcn_frexp_expf(b);
    return __builtin_amdgcn_ldexpf(sum * __builtin_amdgcn_frexp_mantf(a) * __builtin_amdgcn_frexp_mantf(b), ea + eb);
}
__device__ __forceinline__ float scaled(float sum, float a, float b) { return plain_scale(a) && plain_scale(b) ? sum * a * b : scaled_any(sum, a, b); }

__device__ __forceinline__ v4i mfma(v4i a, v4i b, v4i c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float scale_of(const float *scales, int64_t i, int64_t rows) { return scales && i < rows ? scales[i] : 1.0f; }

// A workgroup of WM x WN waves, FM x FN fragments each: a tile of 16 FM WM rows and 16 FN WN columns.  Steps of 64 along the
// reduction go from memory to one of STAGES places in LDS without passing through registers (the storage is
// what a wavefront's 16-byte loads deliver, lane by lane), and a step's fragments are read into
// registers while the step before is multiplied.
template <int FM, int FN, int WM, int WN, int STAGES> struct Gemm {
    static constexpr int WAVES = WM * WN, AM = FM * WM, BN = FN * WN;                // fragments of a tile's sides
    static constexpr int A = 0, B = AM * 1024, BYTES = B + BN * 1024;
    static constexpr int FROM_A = AM / WAVES, LOADS = (AM + BN) / WAVES;             // loads of a wave for a step
    static constexpr int READS = FM + FN;                                            // of LDS
    struct Registers {
        v4i a[FM], b[FN];
    };
};

template <int FM, int FN, int WM, int WN, int STAGES, int RESIDENT>
__global__ __launch_bounds__(64 * WM * WN, RESIDENT) void gemm_kernel(GemmJobs jobs)
{
    using K = Gemm<FM, FN, WM, WN, STAGES>;
    // (a tile's results go out by way of the same LDS, a corner to a wave)
    constexpr int CORNER = Rows<float, FM, FN>::BYTES > Rows<__bf16, FM, FN>::BYTES ? Rows<float, FM, FN>::BYTES : Rows<__bf16, FM, FN>::BYTES;
    constexpr int LDS = STAGES * K::BYTES > K::WAVES * CORNER ? STAGES * K::BYTES : K::WAVES * CORNER;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[LDS];
    static_assert(K::AM % K::WAVES == 0 && K::BN % K::WAVES == 0, "");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
    const bool other = blockIdx.x >= jobs.blocks;
    const GemmArgs g = jobs.job[other];
    const unsigned id = blockIdx.x - (other ? jobs.blocks : 0), tiles = g.tiles_m * g.tiles_n, split = g.splits > 1 ? id / tiles : 0;
    unsigned tm, tn;
    place_tile(id - split * tiles, g.tiles_m, g.tiles_n, tm, tn);
    const int64_t beg = split * g.steps_per_split, end = min(beg + g.steps_per_split, g.steps);
    const int count = (int)(end - beg);

    // what this wave fetches: fragments of either operand
    const uint8_t *fetch[K::LOADS];
    int to[K::LOADS];
#pragma unroll
    for (int i = 0; i < K::LOADS; ++i) {
        const bool of_a = i < K::FROM_A;
        const int f = of_a ? K::FROM_A * wave + i : (K::LOADS - K::FROM_A) * wave + i - K::FROM_A;
        const Operand &o = of_a ? g.a : g.b;
        const int64_t at = min<int64_t>((of_a ? tm * K::AM : tn * K::BN) + f, o.fragments - 1);
        fetch[i] = o.codes + (at * g.steps + beg) * 1024;
        to[i] = (of_a ? K::A : K::B) + f * 1024;
    }
    auto fetch_step = [&](int s) {
        uint8_t *stage = lds + s % STAGES * K::BYTES;
        const int at = min(s, count - 1);
#pragma unroll
        for (int i = 0; i < K::LOADS; ++i) load_to_lds<16>(fetch[i], at * 1024, stage + to[i]);
    };
    auto read_step = [&](int s, typename K::Registers &r) {
        const uint8_t *stage = lds + s % STAGES * K::BYTES;
#pragma unroll
        for (int i = 0; i < FM; ++i) r.a[i] = *(const v4i *)(stage + K::A + (wm * FM + i) * 1024 + lane * 16);
#pragma unroll
        for (int i = 0; i < FN; ++i) r.b[i] = *(const v4i *)(stage + K::B + (wn * FN + i) * 1024 + lane * 16);
    };
    v4i acc[FM][FN] = {};
    auto multiply = [&](const typename K::Registers &r) {
        for_each<FM * FN>([&](auto at) {
            constexpr int i = at.value / FN, j = at.value % FN;
            acc[i][j] = mfma(r.b[j], r.a[i], acc[i][j]);
        });
    };
    // One step: everyone has read step s and its successor's loads are in LDS; loads of step s + STAGES take the
    // place of step s; fragments of s + 1 are read while those of s are multiplied.  (Without branches, so that the
    // multiplications stay where they are: behind the last step it is loaded again, and not used.)
    auto step = [&](int s, const typename K::Registers &now, typename K::Registers &next) {
        AMSIM_WAIT_LDS();
        AMSIM_WAIT_LOADS((STAGES - 2) * K::LOADS);
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
    AMSIM_WAIT_LOADS((STAGES - 1) * K::LOADS);
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
    AMSIM_WAIT_LDS();
    AMSIM_WAIT_LOADS(0);
    meet();  // (LDS is free)
    const int64_t m0 = (int64_t)(tm * WM + wm) * FM * 16, n0 = (int64_t)(tn * WN + wn) * FN * 16;
    if (m0 >= g.a.rows || n0 >= g.b.rows) return;
    uint8_t *mine = lds + wave * CORNER;
    if (g.partial) {
        store_tile<int, FM, FN>(mine, [&](int i, int j, int e) { return acc[i][j][e]; }, g.partial + split * g.a.rows * g.b.rows, m0, n0, g.a.rows, g.b.rows, false);
        return;
    }
    float bias[FN][4], sb[FN][4], sa[FM];
#pragma unroll
    for (int i = 0; i < FM; ++i) sa[i] = scale_of(g.a.scales, m0 + 16 * i + lane % 16, g.a.rows);
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t n = n0 + 16 * j + lane / 16 * 4 + e;
            sb[j][e] = scale_of(g.b.scales, n, g.b.rows);
            bias[j][e] = g.bias && n < g.b.rows ? load_as_float(g.bias, g.bias_dtype, n) : 0.0f;
        }
    bool plain = true;
#pragma unroll
    for (int i = 0; i < FM; ++i) plain = plain && plain_scale(sa[i]);
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) plain = plain && plain_scale(sb[j][e]);
    plain = __all(plain);
    auto store = [&](auto zero, auto *out) {
        using T = decltype(zero);
        auto tile = [&](auto &&scale) {
            store_tile<T, FM, FN>(mine, [&](int i, int j, int e) { return from_float<T>(activate(scale((float)acc[i][j][e], sa[i], sb[j][e]) + bias[j][e], g.act)); }, out,
                                  m0, n0, g.a.rows, g.b.rows, g.around);
        };
        if (plain) tile([](float sum, float a, float b) { return sum * a * b; });
        else tile([](float sum, float a, float b) { return scaled_any(sum, a, b); });
    };
    if (g.out_dtype == AMSIM_DTYPE_F32) store(0.0f, (float *)g.out);
    else if (g.out_dtype == AMSIM_DTYPE_BF16) store((__bf16)0.0f, (__bf16 *)g.out);
    else store((_Float16)0.0f, (_Float16 *)g.out);
}

// Few rows: bound by the reading of b, and for one layer of one token by latency alone.  A workgroup takes 16
// of b's rows and the whole reduction, its waves every n-th step each; their sums meet in LDS.
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
    __device__ __forceinline__ void load(const FewArgs &g, int64_t f, int64_t s, int waves)
    {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) {
            const int64_t t = min<int64_t>(s + h * waves, g.steps - 1);
            codes[h] = *(const v4i *)(g.b.codes + ((f * g.steps + t) * 64 + lane) * 16);
        }
    }
};

// What the results are scaled by and added to, under way since the kernel's start: behind the sums each would be another
// round trip to memory.
struct FewEnds {
    float scale[4], bias[4];
    __device__ __forceinline__ void load(const FewArgs &g, int64_t f)
    {
        const int64_t n = f * 16 + (threadIdx.x & 63) / 16 * 4, N = g.b.rows;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            scale[e] = scale_of(g.b.scales, n + e, N);
            bias[e] = g.bias && n + e < N ? load_as_float(g.bias, g.bias_dtype, n + e) : 0.0f;
        }
    }
};

// the fragments' sums over the waves and their results, a fragment to a wave; row_scales: of the rows, in LDS or memory
template <int FA>
__device__ __forceinline__ void finish_few(const FewArgs &g, const FewEnds &ends, int64_t f, v4i *sums, const v4i (&acc)[FA], const float *row_scales)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int64_t n = f * 16 + lane / 16 * 4, N = g.b.rows;
    float sa[FA];
    bool plain = true;
#pragma unroll
    for (int i = 0; i < FA; ++i) sa[i] = scale_of(row_scales, 16 * i + lane % 16, g.rows), plain = plain && plain_scale(sa[i]);
#pragma unroll
    for (int e = 0; e < 4; ++e) plain = plain && plain_scale(ends.scale[e]);
    plain = __all(plain);
#pragma unroll
    for (int i = 0; i < FA; ++i) sums[(wave * FA + i) * 64 + lane] = acc[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < FA; ++i) {
        if (i % waves != wave) continue;
        v4i z = sums[i * 64 + lane];
        for (int w = 1; w < waves; ++w) z += sums[(w * FA + i) * 64 + lane];
        const int64_t m = 16 * i + lane % 16;
        if (m >= g.rows || n >= N) continue;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (plain ? (float)z[e] * sa[i] * ends.scale[e] : scaled_any((float)z[e], sa[i], ends.scale[e])) + ends.bias[e];
        finish4(nullptr, 0, g.act, g.out, g.out_dtype, m, n, N, v);
    }
}

// FA fragments of converted rows.
template <int FA>
__global__ __launch_bounds__(1024) void few_kernel(FewArgs g)
{
    __shared__ v4i sums[16 * FA * 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    FewEnds ends;
    ends.load(g, blockIdx.x);
    v4i acc[FA] = {};
    for (int64_t s = wave; s < g.steps; s += AHEAD * waves) {
        FewSteps b;
        b.load(g, blockIdx.x, s, waves);
        // The rows' codes with them, all at once: a step's loads in their turn would each be a trip to the L2 (64 rows by
        // 4096 x 4096 took 9.5 us that way and take 7.8 this; 16 rows 5.5 either way).
        v4i a[AHEAD][FA];
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) {
            const int64_t t = min<int64_t>(s + h * waves, g.steps - 1);
#pragma unroll
            for (int i = 0; i < FA; ++i) a[h][i] = *(const v4i *)(g.a.codes + ((min<int64_t>(i, g.a.fragments - 1) * g.steps + t) * 64 + lane) * 16);
        }
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) {
            if (s + h * waves >= g.steps) break;
            for_each<FA>([&](auto i) { acc[i.value] = mfma(b.codes[h], a[h][i.value], acc[i.value]); });
        }
    }
    finish_few(g, ends, blockIdx.x, sums, acc, g.a.scales);
}

// FA fragments of rows as they come: every workgroup converts them for itself, into LDS, while its first loads of b are
// under way.  Its threads take the rows' pieces of 8 values in turn and hold them between the search for the largest,
// which meets in LDS (a step is 8 pieces, so that 8 neighbouring lanes are of one row), and the codes.
constexpr int64_t RAW_VALUES = 32768;  // rows x length (in whole steps) that it converts
template <typename X, int FA>
__global__ __launch_bounds__(FA == 4 ? 512 : 1024) void raw_kernel(FewArgs g)
{
    constexpr int HELD = FA == 4 ? 8 : 4;  // pieces of a thread: what RAW_VALUES come to; if there are more they are read again
    extern __shared__ __attribute__((aligned(16))) uint8_t converted[];  // codes [16 values][row][16 bytes]; then the sums
    __shared__ uint32_t largest[16 * FA];
    __shared__ float row_scales[16 * FA];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int rows = (int)g.rows, apart = rows | 1, pieces = (int)g.steps * 8;  // (an odd distance: a row's 16 values lie in different banks)
    FewSteps b;
    b.load(g, blockIdx.x, wave, waves);
    FewEnds ends;
    ends.load(g, blockIdx.x);
    const int down = blockDim.x / pieces, across = blockDim.x % pieces, row0 = threadIdx.x / pieces, at0 = threadIdx.x % pieces;
    struct Piece {
        int row, at;
    };
    auto next = [&](Piece &p) {
        p.row += down, p.at += across;
        if (p.at >= pieces) p.at -= pieces, ++p.row;
    };
    auto load = [&](Piece p, X (&v)[8]) {
        const int64_t count = p.row < rows ? g.k - 8 * p.at : 0;
        const X *x = (const X *)g.x + p.row * g.row_stride + 8 * p.at;
#pragma unroll
        for (int h = 0; h < 8; h += PIECE<X>) {
            const v4i raw = load_piece(x + h, count - h);
            __builtin_memcpy(&v[h], &raw, 16);
        }
    };
    auto look = [&](Piece p, const X (&v)[8]) {
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max(m, magnitude_bits(to_float(v[e])));
        float f = __uint_as_float(m);
        f = with_dpp<MaxOf, 0xb1>(f);
        f = with_dpp<MaxOf, 0x4e>(f);
        f = with_dpp<MaxOf, 0x141>(f);
        if (lane % 8 == 0 && p.row < rows) atomicMax(&largest[p.row], __float_as_uint(f));  // (of LDS; the largest of any order)
    };
    auto store = [&](Piece p, const X (&v)[8]) {
        if (p.row >= rows) return;
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = to_float(v[e]);
        store_codes(converted + (p.at / 2 * apart + p.row) * 16 + p.at % 2 * 8, f, q8_multiplier(largest[p.row]));
    };
    X held[HELD][8];
    Piece piece{row0, at0};
#pragma unroll
    for (int j = 0; j < HELD; ++j, next(piece)) load(piece, held[j]);
    const Piece rest = piece;  // behind what is held
    if (threadIdx.x < 16 * FA) largest[threadIdx.x] = 0;
    __syncthreads();
    piece = {row0, at0};
#pragma unroll
    for (int j = 0; j < HELD; ++j, next(piece)) look(piece, held[j]);
    // (all lanes of a wave go round: its neighbours' maxima are read across lanes)
    for (Piece p = rest; __any(p.row < rows); next(p)) {
        X v[8];
        load(p, v);
        look(p, v);
    }
    __syncthreads();
    if (threadIdx.x < rows) row_scales[threadIdx.x] = q8_scale(largest[threadIdx.x]);
    piece = {row0, at0};
#pragma unroll
    for (int j = 0; j < HELD; ++j, next(piece)) store(piece, held[j]);
    for (Piece p = rest; p.row < rows; next(p)) {
        X v[8];
        load(p, v);
        store(p, v);
    }
    __syncthreads();
    int row[FA];
#pragma unroll
    for (int i = 0; i < FA; ++i) row[i] = min(16 * i + lane % 16, rows - 1);  // (results of rows that do not exist are not stored)
    v4i acc[FA] = {};
    for (int64_t s = wave; s < g.steps; s += AHEAD * waves) {
        if (s != wave) b.load(g, blockIdx.x, s, waves);
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) {
            const int t = (int)s + h * waves;
            if (t >= g.steps) break;
#pragma unroll
            for (int i = 0; i < FA; ++i) acc[i] = mfma(b.codes[h], *(const v4i *)(converted + ((4 * t + lane / 16) * apart + row[i]) * 16), acc[i]);
        }
    }
    __syncthreads();  // (the sums take the place of what was converted)
    finish_few(g, ends, blockIdx.x, (v4i *)converted, acc, row_scales);
}

// The sums of split reductions, added in 64 bits (2 x 512 x 512 4.0 us: a launch).
constexpr int FINISH_WG = 256;
struct FinishArgs {
    GemmJobs products;
    unsigned blocks[2];      // of either product's sums
};
__global__ __launch_bounds__(FINISH_WG) void finish_kernel(FinishArgs f)
{
    unsigned id = blockIdx.x;
    const bool other = id >= f.blocks[0];
    if (other) id -= f.blocks[0];
    const GemmArgs &g = f.products.job[other];
    const int64_t N = g.b.rows, quads = ceil_div64(N, 4), at = (int64_t)id * FINISH_WG + threadIdx.x;
    if (at >= g.a.rows * quads) return;
    const int64_t m = at / quads, n = at % quads * 4;
    const int count = (int)(N - n < 4 ? N - n : 4);
    const int *p = g.partial + m * N + n;
    const int64_t apart = g.a.rows * N;
    v4i part[MOST_SPLITS];  // (all under way at once: one after the other they take a microsecond each)
#pragma unroll
    for (int s = 0; s < MOST_SPLITS; ++s) {
        part[s] = v4i{0, 0, 0, 0};
        if (s >= g.splits) continue;
        if (count == 4) {
            part[s] = load16(p + s * apart);
        } else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (i < count) part[s][i] = p[s * apart + i];
        }
    }
    const float sa = scale_of(g.a.scales, m, g.a.rows);
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        int64_t z = 0;
#pragma unroll
        for (int s = 0; s < MOST_SPLITS; ++s) z += part[s][i];
        v[i] = scaled((float)(double)z, sa, scale_of(g.b.scales, n + i, N));  // (exact in 64 bits, rounded once)
    }
    finish4(g.bias, g.bias_dtype, g.act, g.out, g.out_dtype, m, n, N, v);
}

// As the 4-bit products': a step is as many bytes and as long on the matrix units.  Over twenty shapes of 100 to 8192 rows, 300 to
// 8192 columns and lengths of 128 to 16384 the choice takes at most 1.12 times the best tile's time, 1.02 on average.  Tiles of
// 256 x 256 in waves of 128 x 64 results: 4096^3 54.5 us (2.5 POP/s), in waves of 64 x 128 55.2, of 128 x 128 (four waves) 69; 8192^3 395
// (2.8; the instruction alone, from registers, runs at 3.5 on random operands, which the card's power allows, and at 4.6 on zeros).
struct Costs {
    static constexpr Tile TILES[] = {{256, 256, 256, 2.2, 0.55, 0.785, 10.8},  // (stored by a round at once)
                                     {256, 128, 512, 6.5, 0.5, 0.85, 0.0124}, {128, 128, 512, 5, 0.2, 0.46, 0.01}, {64, 64, 1024, 4, 0.1, 0.4, 0.003}};
    static constexpr int64_t STEP = I8_STEP, MOST_STEPS = I8_MOST_STEPS;
};

// Whether few_kernel serves: a reduction beyond that needs more than one workgroup's waves, and a wider result has every workgroup
// fetch the rows again for 16 columns.  us of the product by itself, few_kernel / tiles, of 16, 32 and 64 rows:
//   length 1024    8192 wide 4.8/5.2, 5.4/5.6, 6.2/6.1       32768 wide 12.2/9.5, 15.1/9.7, -
//   length 4096    4096 wide 5.5/10.2, 6.9/10.7, 7.8/11.6    8192 wide 8.3/11.7, 8.7/11.7, 11.2/11.7    32768 wide 32.9/28.8, 38.7/30.7, 51.0/30.9
//   length 8192    1024 wide 6.2/12.2, 7.6/10.7, 10.1/11.9   8192 wide 13.3/16.6, 13.9/17.0, 18.2/17.9
//   length 16384   1024 wide 8.9/14.4, 11.2/15.1, 17.4/15.4  4096 wide 12.7/17.6, 13.9/18.3, 19.1/18.9  8192 wide 34.4/41.8, 39.8/42.5, 51.2/43.5
// The three bounds take the quicker up to 32 rows, and of 64 up to a length of 8192 (within 2 %); 64 rows of the longest take up to
// 1.18 times as long as in tiles.
bool few(const Extents &e) { return e.m <= 64 && e.n <= 8192 && i8_steps(e.k) <= 256; }

// the products of a list that go in tiles, and the others
int tiled(const Extents *e, int count, Extents *out, int *which)
{
    int n = 0;
    for (int j = 0; j < count; ++j)
        if (!few(e[j])) out[n] = e[j], which[n++] = j;
    return n;
}

size_t products_workspace(const Extents *e, int count)
{
    Extents t[2];
    int which[2];
    const int n = tiled(e, count, t, which);
    if (n == 0) return 0;
    const Plan p = plan<Costs>(t, n);
    size_t bytes = 0;
    for (int j = 0; j < n; ++j) bytes += partial_bytes(t[j], p.of[j].splits);
    return bytes;
}
size_t product_workspace(int64_t m, int64_t n, int64_t k)
{
    const Extents e{m, n, k};
    return products_workspace(&e, 1);
}

int launch_few(void (*kernel)(FewArgs), const FewArgs &g, int waves, int64_t lds, hipStream_t stream)
{
    if (g.b.fragments >= (1ll << 22)) return fail(AMSIM_ERR_UNSUPPORTED, "int8: more tiles than one launch takes");
    kernel<<<(unsigned)g.b.fragments, 64 * waves, lds, stream>>>(g);
    AMSIM_HIP_CHECK(hipGetLastError());
    return AMSIM_OK;
}
// A wave for every step, and for 128 of the pieces of 8 values that are to be converted first.  Eight waves for up to four rows
// (calls in a row, us: one token of 4096 x 4096 6.8, 7.3 with sixteen; of 8192 x 8192 13.6 and 15.7), sixteen for more (8 rows: 8.5,
// 10.1 with eight).
int few_waves(const FewArgs &g, int64_t pieces)
{
    const int most = g.rows <= 4 ? 8 : 16;
    int waves = 1;
    while (waves < most && (waves < g.steps || 128 * waves < pieces)) waves *= 2;
    return waves;
}
template <typename X> int launch_raw(const FewArgs &g, hipStream_t stream)
{
    // (eight waves' sums of four fragments are 32 KB of LDS, sixteen waves' with the rest would be more than 64)
    const int fragments = g.rows <= 16 ? 1 : g.rows <= 32 ? 2 : 4, waves = std::min(few_waves(g, g.rows * g.steps * 8), fragments == 4 ? 8 : 16);
    const int64_t lds = std::max<int64_t>(g.steps * 4 * (g.rows | 1) * 16, waves * fragments * 1024);
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

// One or two products.
int products(const Product *list, int count, void *workspace, hipStream_t stream)
{
    Extents e[2], t[2];
    int which[2];
    for (int j = 0; j < count; ++j) e[j] = {list[j].a.rows, list[j].b.rows, list[j].k};
    const int n = tiled(e, count, t, which);
    for (int j = 0; j < count; ++j) {
        const Product &q = list[j];
        if (!few(e[j])) continue;
        const FewArgs f{q.b, q.a, nullptr, 0, q.a.rows, q.k, i8_steps(q.k), q.bias, q.bias_dtype, q.act, q.out_dtype, q.out};
        if (int rc = launch_few(q.a.rows <= 16 ? few_kernel<1> : q.a.rows <= 32 ? few_kernel<2> : few_kernel<4>, f, few_waves(f, 0), 0, stream)) return rc;
    }
    if (!n) return AMSIM_OK;
    Plan p = plan<Costs>(t, n);
    if (n == 2 && p.of[1].steps_per_split > p.of[0].steps_per_split)  // the tiles that take longest go first
        std::swap(t[0], t[1]), std::swap(which[0], which[1]), std::swap(p.of[0], p.of[1]);
    FinishArgs f{};
    GemmJobs &jobs = f.products;
    int64_t blocks = 0;
    char *partial = (char *)workspace;
    for (int j = 0; j < n; ++j) {
        const Product &q = list[which[j]];
        const auto &o = p.of[j];
        jobs.job[j] = GemmArgs{q.a, q.b, i8_steps(q.k), o.steps_per_split, q.bias, q.bias_dtype, q.act, q.out_dtype, q.out, (unsigned)o.tiles_m,
                               (unsigned)o.tiles_n, (int)o.splits, mx_goes_around((double)t[j].m * (double)t[j].n * element_bytes(q.out_dtype)),
                               o.splits > 1 ? (int *)partial : nullptr};
        partial += partial_bytes(t[j], o.splits);
        if (j == 0) jobs.blocks = (unsigned)std::min<int64_t>(o.tiles_m * o.tiles_n * o.splits, 1 << 30);
        blocks += o.tiles_m * o.tiles_n * o.splits;
        if (o.splits > 1) f.blocks[j] = (unsigned)ceil_div64(t[j].m * ceil_div64(t[j].n, 4), FINISH_WG);
        // (a launch has less than 2^32 threads)
        if (blocks >= (1ll << 22) || (o.splits > 1 && ceil_div64(t[j].m * ceil_div64(t[j].n, 4), FINISH_WG) >= (1ll << 23)))
            return fail(AMSIM_ERR_UNSUPPORTED, "int8: more tiles than one launch takes");
    }
    switch (p.tile) {
    case 0: gemm_kernel<8, 4, 2, 4, 4, 2><<<(unsigned)blocks, 512, 0, stream>>>(jobs); break;
    case 1: gemm_kernel<8, 4, 2, 2, 3, 2><<<(unsigned)blocks, WG, 0, stream>>>(jobs); break;
    case 2: gemm_kernel<4, 4, 2, 2, 4, 2><<<(unsigned)blocks, WG, 0, stream>>>(jobs); break;
    default: gemm_kernel<2, 2, 2, 2, 4, 4><<<(unsigned)blocks, WG, 0, stream>>>(jobs); break;
    }
    AMSIM_HIP_CHECK(hipGetLastError());
    if (const unsigned last = f.blocks[0] + f.blocks[1]) {
        finish_kernel<<<last, FINISH_WG, 0, stream>>>(f);
        AMSIM_HIP_CHECK(hipGetLastError());
    }
    return AMSIM_OK;
}
int product(const Product &q, void *workspace, hipStream_t stream) { return products(&q, 1, workspace, stream); }

bool product_fits(int64_t m, int64_t n, int64_t k) { return i8_extents_fit(m, k) && i8_extents_fit(n, k) && mx_extents_fit(m, n) && m && n && k; }

int check_product(int64_t m, int64_t n, int64_t k, const void *bias, int bias_dtype, int act, const void *out, int out_dtype)
{
    if (!known_dtype(out_dtype) || (bias && !known_dtype(bias_dtype))) return fail(AMSIM_ERR_INVALID, "int8: unknown element type");
    if (act != AMSIM_ACT_NONE && act != AMSIM_ACT_RELU) return fail(AMSIM_ERR_INVALID, "int8: unknown activation");
    if (!i8_extents_fit(m, k) || !i8_extents_fit(n, k) || !mx_extents_fit(m, n)) return fail(AMSIM_ERR_UNSUPPORTED, "int8: extents out of range");
    if (m == 0 || n == 0 || k == 0) return fail(AMSIM_ERR_INVALID, "int8: empty product");
    if (!out) return fail(AMSIM_ERR_INVALID, "int8: null pointer");
    if ((uintptr_t)out & 15) return fail(AMSIM_ERR_INVALID, "int8: misaligned pointer");
    if (bias && ((uintptr_t)bias & (element_bytes(bias_dtype) - 1))) return fail(AMSIM_ERR_INVALID, "int8: misaligned pointer");
    return AMSIM_OK;
}
int check_workspace(const void *workspace, size_t have, size_t need)
{
    if (need && (!workspace || have < need || ((uintptr_t)workspace & 255))) return fail(AMSIM_ERR_WORKSPACE, "int8: workspace missing, misaligned or too small");
    return AMSIM_OK;
}

// Whether few rows are converted by every workgroup that multiplies them, not once ahead, by a launch more of the device and of
// the host.  us so, and ahead, calls in a row: one token of 4096 x 4096 6.8 and 9.3, 4 rows 7.2 and 9.0, 8 rows 8.7 and 8.9; one of
// 8192 x 8192 13.8 and 15.6; 13 rows of 2051 x 1003 in 32 bits 7.2 and 7.7; 24 rows of 224 x 54 6.0 and 7.6, 32 rows of 1024 x 1024 7.4 and
// 8.4, of 1024 x 4096 7.9 and 8.0, 64 rows of 512 x 512 8.0 and 7.7, of 512 x 4096 8.3 and 7.8.
bool converts_on_the_way(int64_t m, int64_t n, int64_t k) { return m <= 64 && m * i8_steps(k) * I8_STEP * ceil_div64(n, 4096) <= RAW_VALUES; }

size_t aligned(int64_t bytes) { return ((size_t)bytes + 255) / 256 * 256; }
size_t operand_bytes(int64_t rows, int64_t length) { return aligned(i8_bytes(rows, length)); }
// what a training step keeps: an operand's codes, and the scales of the other axis
size_t kept_bytes(int64_t rows, int64_t length) { return (size_t)(i8_code_bytes(rows, length) + 4 * length); }
const float *kept_scales(const void *kept, int64_t rows, int64_t length) { return (const float *)((const uint8_t *)kept + i8_code_bytes(rows, length)); }

}  // namespace

}  // namespace amsim

using namespace amsim;

extern "C" {

int amsim_i8_plan(int count, const int64_t *extents, int64_t *info)
{
    if (count < 1 || count > 2 || !extents || !info) return fail(AMSIM_ERR_INVALID, "int8: one or two products are planned");
    Extents e[2], t[2];
    int which[2];
    for (int j = 0; j < count; ++j) {
        e[j] = {extents[3 * j], extents[3 * j + 1], extents[3 * j + 2]};
        if (!product_fits(e[j].m, e[j].n, e[j].k)) return fail(AMSIM_ERR_UNSUPPORTED, "int8: extents out of range");
    }
    info[0] = info[1] = info[2] = info[3] = 0;
    if (const int n = tiled(e, count, t, which)) {
        const Plan p = plan<Costs>(t, n);
        info[0] = Costs::TILES[p.tile].rows, info[1] = Costs::TILES[p.tile].cols;
        for (int j = 0; j < n; ++j) info[2 + which[j]] = p.of[j].splits;
    }
    return AMSIM_OK;
}

size_t amsim_i8_matmul_workspace_bytes(int64_t m, int64_t n, int64_t k) { return product_fits(m, n, k) ? product_workspace(m, n, k) : 0; }

int amsim_i8_matmul(const void *a, const void *b, int64_t m, int64_t n, int64_t k, const void *bias, int bias_dtype, int act, void *out,
                    int out_dtype, void *workspace, size_t workspace_bytes, void *stream)
{
    if (int rc = check_product(m, n, k, bias, bias_dtype, act, out, out_dtype)) return rc;
    if (!a || !b) return fail(AMSIM_ERR_INVALID, "int8: null pointer");
    if (((uintptr_t)a & 15) || ((uintptr_t)b & 15)) return fail(AMSIM_ERR_INVALID, "int8: misaligned pointer");
    if (int rc = check_workspace(workspace, workspace_bytes, product_workspace(m, n, k))) return rc;
    return product({operand(a, m, k), operand(b, n, k), k, bias, bias_dtype, act, out, out_dtype}, workspace, (hipStream_t)stream);
}

size_t amsim_i8_linear_workspace_bytes(int64_t m, int64_t n, int64_t k)
{
    if (!product_fits(m, n, k) || converts_on_the_way(m, n, k)) return 0;
    return operand_bytes(m, k) + product_workspace(m, n, k);
}

int amsim_i8_linear(const void *x, int dtype, int64_t row_stride, const void *w, int64_t m, int64_t n, int64_t k, const void *bias,
                    int bias_dtype, int act, void *out, void *workspace, size_t workspace_bytes, void *stream)
{
    if (int rc = check_product(m, n, k, bias, bias_dtype, act, out, dtype)) return rc;
    if (!x || !w) return fail(AMSIM_ERR_INVALID, "int8: null pointer");
    if (row_stride < k && m > 1) return fail(AMSIM_ERR_INVALID, "int8: rows overlap");
    if (((uintptr_t)x & (element_bytes(dtype) - 1)) || ((uintptr_t)w & 15)) return fail(AMSIM_ERR_INVALID, "int8: misaligned pointer");
    if (int rc = check_workspace(workspace, workspace_bytes, amsim_i8_linear_workspace_bytes(m, n, k))) return rc;
    if (converts_on_the_way(m, n, k)) {
        const FewArgs f{operand(w, n, k), {}, x, row_stride, m, k, i8_steps(k), bias, bias_dtype, act, dtype, out};
        switch (dtype) {
        case AMSIM_DTYPE_F32: return launch_raw<float>(f, (hipStream_t)stream);
        case AMSIM_DTYPE_BF16: return launch_raw<__bf16>(f, (hipStream_t)stream);
        default: return launch_raw<_Float16>(f, (hipStream_t)stream);
        }
    }
    uint8_t *codes = (uint8_t *)workspace;
    float *scales = (float *)(codes + i8_code_bytes(m, k));
    const I8Rows job{x, nullptr, dtype, m, k, row_stride, nullptr, codes, nullptr, scales};
    if (int rc = i8_convert(&job, nullptr, nullptr, (hipStream_t)stream)) return rc;
    return product({operand(codes, scales, m), operand(w, n, k), k, bias, bias_dtype, act, out, dtype}, codes + operand_bytes(m, k), (hipStream_t)stream);
}

size_t amsim_i8_kept_workspace_bytes(int64_t rows, int64_t length) { return i8_extents_fit(rows, length) && rows && length ? kept_bytes(rows, length) : 0; }

size_t amsim_i8_dense_workspace_bytes(int64_t m, int64_t n, int64_t k)
{
    return product_fits(m, n, k) ? operand_bytes(m, k) + operand_bytes(n, k) + aligned(4 * i8_partial_floats(k, n)) + product_workspace(m, n, k) : 0;
}

int amsim_i8_dense(const void *x, int dtype, int64_t row_stride, const void *kernel, int kernel_dtype, int64_t kernel_row_stride,
                   int64_t m, int64_t n, int64_t k, const void *bias, int bias_dtype, int act, void *out, void *x_kept,
                   void *kernel_kept, void *workspace, size_t workspace_bytes, void *stream)
{
    if (int rc = check_product(m, n, k, bias, bias_dtype, act, out, dtype)) return rc;
    if (!known_dtype(kernel_dtype)) return fail(AMSIM_ERR_INVALID, "int8: unknown element type");
    if ((x_kept && !i8_extents_fit(k, m)) || (kernel_kept && !i8_extents_fit(k, n))) return fail(AMSIM_ERR_UNSUPPORTED, "int8: extents out of range");
    if (!x || !kernel) return fail(AMSIM_ERR_INVALID, "int8: null pointer");
    if ((row_stride < k && m > 1) || (kernel_row_stride < n && k > 1)) return fail(AMSIM_ERR_INVALID, "int8: rows overlap");
    if (((uintptr_t)x & (element_bytes(dtype) - 1)) || ((uintptr_t)kernel & (element_bytes(kernel_dtype) - 1)) || ((uintptr_t)x_kept & 15)
        || ((uintptr_t)kernel_kept & 15))
        return fail(AMSIM_ERR_INVALID, "int8: misaligned pointer");
    if (int rc = check_workspace(workspace, workspace_bytes, amsim_i8_dense_workspace_bytes(m, n, k))) return rc;
    hipStream_t s = (hipStream_t)stream;
    uint8_t *x_rows = (uint8_t *)workspace, *kernel_columns = x_rows + operand_bytes(m, k);
    float *looked = (float *)(kernel_columns + operand_bytes(n, k));
    void *partial = (uint8_t *)looked + aligned(4 * i8_partial_floats(k, n));
    // (where they are kept, the scales lie with the codes that are)
    float *x_scales = x_kept ? (float *)kept_scales(x_kept, k, m) : (float *)(x_rows + i8_code_bytes(m, k));
    float *kernel_scales = kernel_kept ? (float *)kept_scales(kernel_kept, k, n) : (float *)(kernel_columns + i8_code_bytes(n, k));
    const I8Rows rows{x, nullptr, dtype, m, k, row_stride, nullptr, x_rows, (uint8_t *)x_kept, x_scales};
    const I8Columns columns{kernel, nullptr, kernel_dtype, k, n, kernel_row_stride, nullptr, (uint8_t *)kernel_kept, kernel_columns, kernel_scales, nullptr, 0};
    if (int rc = i8_convert(&rows, &columns, looked, s)) return rc;
    return product({operand(x_rows, x_scales, m), operand(kernel_columns, kernel_scales, n), k, bias, bias_dtype, act, out, dtype}, partial, s);
}

static size_t gradient_columns_bytes(int64_t m, int64_t n, int64_t k) { return i8_extents_fit(k, m) ? operand_bytes(n, m) : 0; }

size_t amsim_i8_dense_grad_workspace_bytes(int64_t m, int64_t n, int64_t k)
{
    if (!product_fits(m, n, k)) return 0;
    // (the products of either gradient alone are planned by themselves, and one whose reduction is too long is not asked for)
    const Extents e[2] = {{m, k, n}, {k, n, m}};
    const bool of_x = i8_extents_fit(k, n), of_kernel = i8_extents_fit(k, m);
    return operand_bytes(m, n) + gradient_columns_bytes(m, n, k) + aligned(4 * i8_partial_floats(m, n))
         + std::max({of_x && of_kernel ? products_workspace(e, 2) : 0, of_x ? products_workspace(e, 1) : 0, of_kernel ? products_workspace(e + 1, 1) : 0});
}

int amsim_i8_dense_grad(const void *grad, int dtype, int64_t row_stride, const void *out, const void *x_kept, const void *kernel_kept,
                        int64_t m, int64_t n, int64_t k, void *grad_x, void *grad_kernel, int kernel_dtype, void *grad_bias, int bias_dtype,
                        void *workspace, size_t workspace_bytes, void *stream)
{
    if (!known_dtype(dtype) || (grad_kernel && !known_dtype(kernel_dtype)) || (grad_bias && !known_dtype(bias_dtype)))
        return fail(AMSIM_ERR_INVALID, "int8: unknown element type");
    if (!i8_extents_fit(m, k) || !i8_extents_fit(n, k) || !mx_extents_fit(m, n) || (grad_x && !i8_extents_fit(k, n)) || (grad_kernel && !i8_extents_fit(k, m)))
        return fail(AMSIM_ERR_UNSUPPORTED, "int8: extents out of range");
    if (m == 0 || n == 0 || k == 0) return fail(AMSIM_ERR_INVALID, "int8: empty product");
    if (row_stride < n && m > 1) return fail(AMSIM_ERR_INVALID, "int8: rows overlap");
    if (!grad || (grad_x && !kernel_kept) || (grad_kernel && !x_kept)) return fail(AMSIM_ERR_INVALID, "int8: null pointer");
    const uintptr_t element = element_bytes(dtype) - 1;
    if (((uintptr_t)grad & element) || ((uintptr_t)out & element) || ((uintptr_t)x_kept & 15) || ((uintptr_t)kernel_kept & 15)
        || ((uintptr_t)grad_x & 15) || ((uintptr_t)grad_kernel & 15) || (grad_bias && ((uintptr_t)grad_bias & (element_bytes(bias_dtype) - 1))))
        return fail(AMSIM_ERR_INVALID, "int8: misaligned pointer");
    if (int rc = check_workspace(workspace, workspace_bytes, amsim_i8_dense_grad_workspace_bytes(m, n, k))) return rc;
    if (!grad_x && !grad_kernel && !grad_bias) return AMSIM_OK;
    hipStream_t s = (hipStream_t)stream;
    uint8_t *rows = (uint8_t *)workspace, *columns = rows + operand_bytes(m, n);
    float *looked = (float *)(columns + gradient_columns_bytes(m, n, k));
    void *partial = (uint8_t *)looked + aligned(4 * i8_partial_floats(m, n));
    float *row_scales = (float *)(rows + i8_code_bytes(m, n)), *column_scales = (float *)(columns + i8_code_bytes(n, m));
    // (the gradient's rows are converted with the kernel's scales on its columns, its columns with x's on its rows)
    const I8Rows by_rows{grad, out, dtype, m, n, row_stride, grad_x ? kept_scales(kernel_kept, k, n) : nullptr, rows, nullptr, row_scales};
    const I8Columns by_columns{grad, out, dtype, m, n, row_stride, grad_kernel ? kept_scales(x_kept, k, m) : nullptr, nullptr, grad_kernel ? columns : nullptr,
                               column_scales, grad_bias, bias_dtype};
    if (int rc = i8_convert(grad_x ? &by_rows : nullptr, grad_kernel || grad_bias ? &by_columns : nullptr, looked, s)) return rc;
    Product list[2];
    int count = 0;
    if (grad_x) list[count++] = {operand(rows, row_scales, m), operand(kernel_kept, nullptr, k), n, nullptr, 0, AMSIM_ACT_NONE, grad_x, dtype};
    if (grad_kernel) list[count++] = {operand(x_kept, nullptr, k), operand(columns, column_scales, n), m, nullptr, 0, AMSIM_ACT_NONE, grad_kernel, kernel_dtype};
    return count ? products(list, count, partial, s) : AMSIM_OK;
}

}  // extern "C"
