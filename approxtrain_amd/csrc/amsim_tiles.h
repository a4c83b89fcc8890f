// What the products on the matrix cores share, whatever they multiply: where a tile lies, steps from memory to LDS, results
// to memory, and the choice of tiles and splits.  A step is what a wavefront's 16 bytes a lane hold of 16 rows: 128 values
// of 4 bits, 64 of 8; it takes the matrix units as long either way.
#ifndef AMSIM_TILES_H_
#define AMSIM_TILES_H_

#include "amsim_mx.h"

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

namespace amsim {

namespace {

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
#define AMSIM_WAIT_LOADS(n) __builtin_amdgcn_s_waitcnt(((n) & 15) | 7 << 4 | 15 << 8 | ((n) >> 4) << 14)
#define AMSIM_WAIT_LDS() __builtin_amdgcn_s_waitcnt(15 | 7 << 4 | 0 << 8 | 3 << 14)
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
    static constexpr int COLUMNS = 16 * FN, STRIDE = COLUMNS * sizeof(T) + 16, AT_ONCE = FM * FN >= 32 ? 32 / FN / sizeof(T) : FM;
    static constexpr int BYTES = 16 * AT_ONCE * STRIDE;
};
// value(i, j, e): of the lane's row in fragment i of the rows, its e-th column in fragment j of the columns.
template <typename T, int FM, int FN, typename Value>
__device__ __forceinline__ void store_tile(uint8_t *lds, Value &&value, T *out, int64_t m0, int64_t n0, int64_t M, int64_t N, bool around)
{
    using R = Rows<T, FM, FN>;
    const int lane = threadIdx.x & 63, columns = (int)min<int64_t>(R::COLUMNS, N - n0);
    for_each<FM / R::AT_ONCE>([&](auto part) {
        constexpr int first = part.value * R::AT_ONCE;
        AMSIM_WAIT_LDS();  // (what lay there before has been read)
        for_each<R::AT_ONCE * FN>([&](auto at) {
            constexpr int i = at.value / FN, j = at.value % FN;
            T t[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = value(first + i, j, e);
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

// ---- the choice of tiles -------------------------------------------------------------------------------------------

constexpr int MOST_SPLITS = 16;
struct Tile {
    int rows, cols, slots;  // slots: tiles that the card holds at once
    // microseconds, as measured on products of 128 to 16384 a side: of a launch; of a step where a tile has a CU for itself,
    // and where all slots are taken; of storing a tile (between results of 16 bits and of 32: workspaces are asked for
    // before the type is known)
    double base, alone, full, store;
};

struct Extents {
    int64_t m, n, k;
};
struct Plan {
    int tile;  // of the list
    struct {
        int64_t tiles_m, tiles_n, splits, steps_per_split;
    } of[2];
};

// What a launch of `tiles` tiles takes whose steps add up to `work` and are at most `longest`: rounds of all slots, and a
// last one in which a CU has one tile or a few.
template <typename Costs> double microseconds(int tile, double tiles, double work, double longest)
{
    const Tile &t = Costs::TILES[tile];
    const double mean = work / tiles, rounds = std::floor(tiles / t.slots), rest = tiles - rounds * t.slots;
    double last = rest > 0 ? std::max(t.alone, t.full * rest / t.slots) : 0;
    if (tile == 1 && rest > 256) last = 0.8;
    const double steps = std::max(rounds * t.full * mean + last * mean, t.alone * longest);
    if (tile == 0) return t.base + std::ceil(tiles / t.slots) * (t.store + 1.5) - 1.5 + steps;
    return t.base + steps + t.store * tiles;
}

// The tile of one or two products and the splits of their reductions that take least time.  A split reduction takes a
// second launch, 3 us, and its sums go to memory and back.  Costs: the list of four TILES, the values of a STEP, and MOST_STEPS that
// one sum may have.
template <typename Costs> Plan make_plan(const Extents *e, int count)
{
    Plan best{-1, {}};
    double least = 0;
    for (int i = 0; i < 4; ++i) {
        Plan p{i, {}};
        double tiles = 0, work = 0, longest = 0, more = 0;
        for (int j = 0; j < count; ++j) {
            const int64_t steps = ceil_div64(e[j].k, Costs::STEP), tiles_m = ceil_div64(e[j].m, Costs::TILES[i].rows), tiles_n = ceil_div64(e[j].n, Costs::TILES[i].cols);
            const double area = (double)tiles_m * (double)tiles_n;
            double quickest = 0, its_more = 0;
            for (int64_t s = 1; s <= MOST_SPLITS && (s == 1 || 2 * s <= steps); s *= 2) {
                const int64_t each = ceil_div64(steps, s), splits = ceil_div64(steps, each);
                const double extra = splits > 1 ? 3 + (double)splits * (double)e[j].m * (double)e[j].n * 8 / 4e6 : 0;
                if (each > Costs::MOST_STEPS) continue;
                const double us = microseconds<Costs>(i, area * splits, area * splits * each, each) + extra;
                if (quickest > 0 && us >= quickest) continue;
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
        const double us = microseconds<Costs>(i, tiles, work, longest) + more;
        if (best.tile < 0 || us < least) {
            least = us;
            best = p;
        }
    }
    return best;
}

// The same, looked up where the thread has asked for it before: a training step asks seven times, a microsecond each.
template <typename Costs> Plan plan(const Extents *e, int count)
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
    if (!same(at.e[0], e[0]) || !same(at.e[1], f)) at = Known{{e[0], f}, make_plan<Costs>(e, count)};
    return at.p;
}

inline size_t partial_bytes(const Extents &e, int64_t splits) { return splits > 1 ? ((size_t)splits * e.m * e.n * 4 + 255) / 256 * 256 : 0; }

}  // namespace

}  // namespace amsim
#endif  // AMSIM_TILES_H_
