#pragma once
// The kernels that products of rows in group order run on matrix cores: tiles of 256 x
// 256, 128 x 128 and 64 x 64, and a kernel for few rows; how one of them is chosen and
// launched.  All take 64 steps of the contraction at a time through LDS.  Many rows are
// bound by how well the matrix cores are fed and by the clock that they leave, few by
// reading the weights.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>
#include <utility>

#include "amdgcn.h"
#include "eight_bits.h"
#include "elements.h"
#include "engine.h"
#include "gated.h"
#include "hip_status.h"

namespace spmm {
namespace engine {
namespace {

using namespace dev;

// A buffer-to-LDS load from a raw buffer (stride 0), in two steps that other
// instructions may come between (none that reads or writes M0): where the load goes,
// then the load of lane i's 16 bytes from byte `offset` to LDS address lds + ADD + 16 i.
// An offset at or past the record count (bytes) writes zeros.  M0 has to be written at
// least one instruction before the load.
template <int ADD>
__device__ __forceinline__ void lds_dma_raw_to(unsigned lds) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    asm volatile("s_add_u32 m0, %0, %1" : : "s"(lds), "n"(ADD) : "m0", "scc");
#pragma clang diagnostic pop
}
__device__ __forceinline__ void lds_dma_raw_x4(u32x4 rsrc, unsigned offset) {
    asm volatile("buffer_load_dwordx4 %0, %1, 0 offen lds" : : "v"(offset), "s"(rsrc));
}

constexpr int kStep = 64;  // contraction steps a staged tile holds
constexpr int kRingLds = 160 * 1024;

// A byte offset past every buffer's 2^31 - 1 bytes, with room for the 16 that a
// load adds: it reads zeros.
constexpr unsigned kAbsent = 0x80000000u;

// A pair of 8-bit integers: rows of them are moved as rows of 16-bit elements, half as
// many, and multiplied by v_mfma_i32_16x16x64_i8, whose operands are as many bytes a lane.
struct Int8Pair {
    signed char low, high;
};
typedef int i32x4 __attribute__((ext_vector_type(4)));

// A 16-bit element type's operand of one 16x16x32 product.
__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ i32x4 mfma(i32x4 a, i32x4 b, i32x4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}
// The same into accumulation registers.  Written out because the compiler moves
// 256 accumulators between the register files instead of leaving them in place.
// What the compiler would count for its own products is kept by the callers: the
// operands come from LDS reads (which it waits for), and the sums are read only
// after settle_sums.
__device__ __forceinline__ void mfma_in_place(f32x4& c, f16x8 a, f16x8 b) {
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
__device__ __forceinline__ void mfma_in_place(f32x4& c, bf16x8 a, bf16x8 b) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
__device__ __forceinline__ void mfma_in_place(i32x4& c, i32x4 a, i32x4 b) {
    asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
// Waits until the last products have left the pipe.  Each sum passes through an
// (empty) statement behind the wait, so that nothing reads it earlier.
template <int CF, int RF, typename V>
__device__ __forceinline__ void settle_sums(V (&acc)[CF][RF]) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
    for (int j = 0; j < CF; ++j)
#pragma unroll
        for (int i = 0; i < RF; ++i) asm volatile("" : "+a"(acc[j][i]));
    __builtin_amdgcn_sched_barrier(0);
}
template <typename T>
using Operand = std::conditional_t<std::is_same_v<T, _Float16>, f16x8,
                                   std::conditional_t<std::is_same_v<T, __bf16>, bf16x8, i32x4>>;
// Four sums: fp32, or of 8-bit integers' products, exact (refused where they could pass 2^31).
template <typename T>
using Sums = std::conditional_t<std::is_same_v<T, Int8Pair>, i32x4, f32x4>;

// What becomes of a tile's sums: they leave as they are (8-bit integers': scaled), with
// their rows' adapters added, as act(g) * u, two columns' sums each, or multiplied by their
// row's or their group's power of two (operands that were held in range by it).
enum class Ends { Plain, Adapters, Gated, Scaled };

struct TileArgs {
    const void* rows;     // X [total, depth], or P [total, height]
    const void* cols;     // W [groups, width, depth] / [groups, depth, width], or Q [total, width]
    void*       out;      // [total, width], or [groups, height, width]
    const int*  offsets;  // groups + 1 first rows; null: one group of all rows
    int         groups;
    int         total;    // rows of X, P, Q
    int         height;   // gradient: rows of each group's output
    int         from, upto; // gradient: those of them that this launch takes
    int         width;    // columns of the output
    int         depth;    // product: contraction
    // adapters (ids null: none)
    const int*  ids;      // total
    const float* h;       // [total, rank16]
    const void* b;        // [adapters, width, rank]
    int         adapters;
    int         rank;
    int         rank16;   // rank rounded up to whole tiles of adapter_shrink
    bool        b_pieces; // B's rows are whole 16-byte pieces
    // gated: W [groups, 2, width, depth], the gates' rows first
    Act         act;
    void*       kept;         // g and u [total, 2, width], of the operands' type or in 8 bits; or null
    unsigned char* kept_scales; // [total, 2, width / 32 rounded up]; null: not in 8 bits
    // 8-bit integers
    const float* row_scales;  // total
    const float* col_scales;  // [groups, width], gated [groups, 2, width]
    ElementType out_type;
    // scaled: row_scales, or in a gradient
    const float* group_scales; // groups
    // where the operands end, for rows that are no whole pieces
    const void* rows_end;
    const void* cols_end;
};

// The group's rows as the kernels use them: in range and in order whatever the
// offsets hold, so that no value of theirs leads outside the operands.
__device__ __forceinline__ int row_bound(const TileArgs& a, int i) {
    if (a.offsets == nullptr) return i == 0 ? 0 : a.total;
    return min(max(a.offsets[i], 0), a.total);
}

// The row tiles of all groups, counted group by group; past the last group come
// the tiles of the rows in no group, those behind the last (group = groups) and
// those before the first (group = groups + 1).  Lane i looks at group i of each 64.
struct RowTile {
    int group, first, end;  // rows [first, end), end <= first + BR; group < 0: no such tile
};
__device__ __forceinline__ void group_rows(const TileArgs& a, int g, int& lo, int& hi) {
    lo = hi = 0;
    if (g <= a.groups) {
        lo = row_bound(a, g);
        hi = g < a.groups ? max(row_bound(a, g + 1), lo) : a.total;
    } else if (g == a.groups + 1) {
        hi = row_bound(a, 0);
    }
}
// Tiles of group g, the first row of the first of them, and the group's end.
template <int BR>
__device__ __forceinline__ int group_tiles(const TileArgs& a, int g, int& lo, int& hi) {
    group_rows(a, g, lo, hi);
    return (hi - lo + BR - 1) / BR;
}
// The tile whose number lies in [upto - tiles, upto) of some lane's group.
template <int BR>
__device__ __forceinline__ bool tile_among(int tile, int g0, int lo, int hi, int tiles, int upto,
                                           RowTile& r) {
    const unsigned long long at = __ballot(tile >= upto - tiles && tile < upto);
    if (at == 0) return false;
    const int l = __builtin_ctzll(at);
    const int first = __shfl(lo + (tile - (upto - tiles)) * BR, l);
    r = RowTile{g0 + l, first, min(first + BR, __shfl(hi, l))};
    return true;
}
// The same for the whole wave, which the compiler does not see.
__device__ __forceinline__ RowTile uniform(RowTile r) {
    return RowTile{__builtin_amdgcn_readfirstlane(r.group), __builtin_amdgcn_readfirstlane(r.first),
                   __builtin_amdgcn_readfirstlane(r.end)};
}
template <int BR>
__device__ __forceinline__ int count_tiles(const TileArgs& a) {
    int tiles = 0;
    for (int g0 = 0; g0 <= a.groups + 1; g0 += 64) {
        int lo, hi;
        const int n = group_tiles<BR>(a, g0 + (threadIdx.x & 63), lo, hi);
        tiles += __shfl(wave_prefix(n), 63);
    }
    return __builtin_amdgcn_readfirstlane(tiles);
}
// A prefix sum over the groups' tiles finds the group that holds `tile`.
template <int BR>
__device__ __forceinline__ RowTile find_tile(const TileArgs& a, int tile) {
    if (a.offsets == nullptr) {
        const int first = tile * BR;
        return first < a.total ? RowTile{0, first, min(first + BR, a.total)} : RowTile{-1, 0, 0};
    }
    RowTile r{-1, 0, 0};
    int before = 0;
    for (int g0 = 0; g0 <= a.groups + 1; g0 += 64) {
        int lo, hi;
        const int tiles = group_tiles<BR>(a, g0 + (threadIdx.x & 63), lo, hi);
        const int upto = before + wave_prefix(tiles);
        if (tile_among<BR>(tile, g0, lo, hi, tiles, upto, r)) break;
        before = __shfl(upto, 63);
    }
    return uniform(r);
}

// The tile of a workgroup: work item w of row_tiles x col_tiles.  Workgroup b
// runs on XCD b mod 8; each XCD takes a contiguous eighth of the items, which go
// through eight row tiles at a time, so that the tiles an XCD works on together
// share their rows and columns in its L2.
__device__ __forceinline__ bool tile_of_block(int row_tiles, int col_tiles, int& rt, int& ct) {
    const long long total = static_cast<long long>(row_tiles) * col_tiles;
    const long long share = (total + 7) / 8;
    const long long local = blockIdx.x >> 3;
    const long long item  = (blockIdx.x & 7) * share + local;
    if (local >= share || item >= total) return false;
    const int band = static_cast<int>(item / (8LL * col_tiles));
    const int rest = static_cast<int>(item - 8LL * col_tiles * band);
    const int high = min(8, row_tiles - 8 * band);
    rt = 8 * band + rest % high;
    ct = rest / high;
    return true;
}

// The row tile and column tile of a workgroup of a product.  Up to 62 groups are
// looked at once, for their number of tiles and for the tile itself.
template <int BR>
__device__ __forceinline__ bool row_tile_of_block(const TileArgs& a, int col_tiles, RowTile& r,
                                                  int& ct) {
    int rt;
    if (a.offsets == nullptr) {
        if (!tile_of_block((a.total + BR - 1) / BR, col_tiles, rt, ct)) return false;
        r = find_tile<BR>(a, rt);
        return true;
    }
    if (a.groups + 2 <= 64) {
        int lo, hi;
        const int tiles = group_tiles<BR>(a, threadIdx.x & 63, lo, hi);
        const int upto = wave_prefix(tiles);
        const int all = __builtin_amdgcn_readfirstlane(__shfl(upto, 63));
        return tile_of_block(all, col_tiles, rt, ct) && tile_among<BR>(rt, 0, lo, hi, tiles, upto, r);
    }
    if (!tile_of_block(count_tiles<BR>(a), col_tiles, rt, ct)) return false;
    r = find_tile<BR>(a, rt);
    return r.group >= 0;
}

// How one operand lies in memory and in LDS.
//   MAJOR false: N rows of the contraction's elements in a row (X, W [c][k]).
//     LDS rows of 64 elements; 16-byte piece p of row n at place p ^ (n & 7), so
//     that the 16 rows of an operand read meet all banks.
//   MAJOR true: the contraction's steps are the rows, N elements each (W [k][c],
//     and both operands of a gradient).  LDS rows of N elements, pieces at place
//     p ^ 2 f(k), f(k) = (k & 3) | ((k >> 3) & 1) << 2: the transposing read of
//     32 lanes takes 32 bytes of rows {0-3, 8-11}, f spreads them over all banks (rows
//     of 64 elements: f(k) = bit 1 | bit 3 << 1, bit 0 being in the address).
//   PARTS 2 (gated products): the first half of the rows and the second half come from
//     two places, as many valid rows each.
template <typename T, int N, bool MAJOR, int THREADS, int PARTS = 1>
struct Operands {
    static constexpr int kPieces = N * kStep / 8 / THREADS;
    static constexpr int kRow    = MAJOR ? N : kStep;  // elements of an LDS row
    static_assert(N * kStep / 8 % THREADS == 0, "whole pieces a thread");
    static_assert(PARTS == 1 || (!MAJOR && kPieces % PARTS == 0), "a piece lies in one part");
    static_assert(!MAJOR || N == 64 || N == 128, "the places of a row are 32 bytes x 4 or 8");

    // f(k), from step k's bits 0, 1 and 3
    static __device__ __forceinline__ int spread(int low, int bit3) {
        return N == 64 ? low >> 1 | bit3 << 1 : low | bit3 << 2;
    }

    unsigned at[kPieces];     // byte offset of the piece from the tile's first word
    int      index[kPieces];  // its first contraction step inside the tile
    int      ld, bound;

    // The tile's first element lies at `first`; ld: elements between memory rows;
    // bound: valid rows (columns for MAJOR), of which there may be more than N.
    __device__ __forceinline__ void place(const T* first, int row_elements, int valid,
                                          const T* second = nullptr) {
        ld    = row_elements;
        bound = valid;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const T* from = PARTS == 2 && i >= kPieces / 2 ? second : first;
            const unsigned odd = static_cast<unsigned>(reinterpret_cast<uintptr_t>(from)) & 2u;
            const int p = i * THREADS + threadIdx.x % THREADS;
            int n, element;
            if constexpr (MAJOR) {
                const int k = p / (N / 8);
                const int f = spread(k & 3, (k >> 3) & 1);
                n        = ((p % (N / 8)) ^ (f << 1)) * 8;
                element  = k * ld + n;
                index[i] = k;
            } else {
                n        = p / 8;
                index[i] = ((p % 8) ^ (n & 7)) * 8;
                if constexpr (PARTS > 1) n = n % (N / PARTS);
                element  = n * ld + index[i];
            }
            at[i] = n < bound ? static_cast<unsigned>(element) * 2u + odd : kAbsent;
        }
    }
    // Loads the tile at `tile` with `left` contraction steps left, in whole words.  The
    // buffer ends with the tile's last valid row, so that no word without an element is
    // read; what a piece holds behind its row's end is cut off by store (MAJOR: it belongs
    // to columns past the bound, which are never stored).  ODD: pieces may begin between
    // two words.
    template <bool ODD>
    __device__ __forceinline__ void load(const T* tile, int left, WordPiece (&v)[kPieces],
                                         const T* second = nullptr) const {
        const long long rows = MAJOR ? min(left, kStep) : min(bound, N / PARTS);
        const __amdgpu_buffer_rsrc_t buffer =
            words_buffer(tile, (rows - 1) * ld + (MAJOR ? bound : left));
        const __amdgpu_buffer_rsrc_t other =
            PARTS == 2 ? words_buffer(second, (rows - 1) * ld + left) : buffer;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            v[i] = load_words<ODD>(PARTS == 2 && i >= kPieces / 2 ? other : buffer,
                                   index[i] < left ? at[i] : kAbsent);
        }
    }
    template <bool ODD>
    __device__ __forceinline__ void store(T* lds, int left, const WordPiece (&v)[kPieces]) const {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            uint4 x = ODD ? piece_of(v[i], at[i]) : v[i].words;
            if constexpr (!MAJOR) {
                if (left < kStep) x = first_of(x, left - index[i]);
            }
            *reinterpret_cast<uint4*>(lds + (i * THREADS + threadIdx.x % THREADS) * 8) = x;
        }
    }
    // Operand of columns n0 .. n0+15, contraction steps 32 half .. +31: lane l holds
    // steps 8 (l >> 4) .. +7 of column l & 15.
    static __device__ __forceinline__ Operand<T> read(const T* lds, int n0, int half) {
        const int lane = threadIdx.x & 63;
        const int q = lane >> 4, s = lane & 15;
        if constexpr (MAJOR) {
            const int k = 32 * half + 8 * q + (s >> 2);
            const int f = spread(s >> 2, q & 1);
            const int c = ((n0 / 16) ^ f) * 16 + (s & 3) * 4;
            const _Float16* p = reinterpret_cast<const _Float16*>(lds) + k * kRow + c;
            const s16x4 x = lds_read_tr16(p);
            const s16x4 y = lds_read_tr16(p + 4 * kRow);
            const s16x8 both = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
            return __builtin_bit_cast(Operand<T>, both);
        } else {
            const int c = (4 * half + q) ^ (s & 7);
            return *reinterpret_cast<const Operand<T>*>(lds + (n0 + s) * kRow + c * 8);
        }
    }
};

// What a workgroup works on: the first elements of its operands and its output,
// the contraction's length, and how far a staged tile advances.
template <typename T>
struct Tile {
    const T* rows;
    const T* cols;
    const T* second;  // gated: the second projection's columns
    T*       out;
    int group, row0, rows_here, c0, depth, ld_rows, ld_cols;
    long long step_rows, step_cols;
};
template <typename T, int BR, int BC, bool GRAD, bool COLS_MAJOR, bool GATED = false>
__device__ __forceinline__ bool take_tile(const TileArgs& a, Tile<T>& t) {
    const int col_tiles = (a.width + BC - 1) / BC;
    t.rows = static_cast<const T*>(a.rows);
    t.cols = static_cast<const T*>(a.cols);
    t.out  = static_cast<T*>(a.out);
    int ct;
    if constexpr (GRAD) {
        int rt;
        const int row_tiles = (a.upto - a.from + BR - 1) / BR;
        if (!tile_of_block(a.groups * row_tiles, col_tiles, rt, ct)) return false;
        const int g = rt / row_tiles;
        t.group = g;
        t.row0 = a.from + (rt % row_tiles) * BR;
        t.rows_here = min(BR, a.upto - t.row0);
        t.c0 = ct * BC;
        const int lo = row_bound(a, g), hi = max(row_bound(a, g + 1), lo);
        t.depth   = hi - lo;
        t.ld_rows = a.height;
        t.ld_cols = a.width;
        t.rows += static_cast<long long>(lo) * t.ld_rows + t.row0;
        t.cols += static_cast<long long>(lo) * t.ld_cols + t.c0;
        t.out  += (static_cast<long long>(g) * a.height + t.row0) * a.width;
        t.step_rows = static_cast<long long>(kStep) * t.ld_rows;
        t.step_cols = static_cast<long long>(kStep) * t.ld_cols;
    } else {
        RowTile r;
        if (!row_tile_of_block<BR>(a, col_tiles, r, ct)) return false;
        r = uniform(r);
        t.row0 = r.first;
        t.rows_here = r.end - r.first;
        t.c0 = ct * BC;
        t.depth   = r.group < a.groups ? a.depth : 0;  // rows in no group: zeros
        t.ld_rows = a.depth;
        t.ld_cols = COLS_MAJOR ? a.width : a.depth;
        t.rows += static_cast<long long>(t.row0) * t.ld_rows;
        t.group = r.group < a.groups ? r.group : 0;
        t.cols += static_cast<long long>(t.group) * (GATED ? 2 : 1) * a.width * a.depth +
                  static_cast<long long>(t.c0) * (COLS_MAJOR ? 1 : t.ld_cols);
        if constexpr (GATED) t.second = t.cols + static_cast<long long>(a.width) * a.depth;
        t.out  += static_cast<long long>(t.row0) * a.width;
        t.step_rows = kStep;
        t.step_cols = COLS_MAJOR ? static_cast<long long>(kStep) * t.ld_cols : kStep;
    }
    return true;
}

// f(0), f(1), ... with the index a constant, so that registers named by it stay
// registers however much f does.
template <int... I, typename F>
__device__ __forceinline__ void unrolled(std::integer_sequence<int, I...>, F f) {
    (f(std::integral_constant<int, I>{}), ...);
}

// Eight values of h as two operands: high + low is h * 2^-shift but for 2^-16 of it
// (bf16) or 2^-22 (fp16), a sixteenth and less of what the result's own rounding takes.
//   shift: brings a row's largest value below 2^14 in fp16, whose range is short of fp32's
//     (bf16 needs none).
//   low is no number where high is not finite.
template <typename T>
struct Parts {
    Operand<T> high, low;
};
template <typename T>
__device__ __forceinline__ Parts<T> parts_of(const float (&v)[8], int shift) {
    T high[8], low[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = std::is_same_v<T, _Float16> ? ldexpf(v[i], -shift) : v[i];
        high[i] = static_cast<T>(x);
        low[i]  = static_cast<T>(x - static_cast<float>(high[i]));
    }
    return Parts<T>{__builtin_bit_cast(Operand<T>, high), __builtin_bit_cast(Operand<T>, low)};
}

// The adapters of a wave's rows (r0 .. of the workgroup's tile, columns c0 ..), added
// sixteen rows at a time on their way out: for each adapter among the rows h against
// B_a, kept only in its own rows, so that no row sees what another's adapter holds,
// infinities and NaN included.
//   PIECES: B's rows are whole 16-byte pieces (buffer loads, 32-bit offsets).
template <typename T, int RF, int CF, bool PIECES>
struct Adapters {
    static constexpr bool kShift = std::is_same_v<T, _Float16>;
    // 32s of the rank whose parts stay for all adapters among sixteen rows (8192 rows x 4096 x
    // 4096, rank 64, an adapter a row: 640 us with two, 685 with one; 701 x 2003 x 1001, rank
    // 12, in 64 x 64 tiles: 32.0 with one, 33.5 with two)
    static constexpr int kKept = CF > 2 ? 2 : 1;
    const float* h;
    const T*     b;
    int          id[RF];     // of row 16 i + (lane & 15), -1 for none
    int          shift[RF];  // of that row's h (kShift only)
    int          width, rank, rank16;
    int          c0;

    __device__ __forceinline__ Adapters(const TileArgs& a, const Tile<T>& t, int r0, int first_col)
        : h(a.h + static_cast<long long>(t.row0 + r0) * a.rank16),
          b(static_cast<const T*>(a.b)), width(a.width), rank(a.rank), rank16(a.rank16),
          c0(first_col) {
        const int s = threadIdx.x & 15;
#pragma unroll
        for (int i = 0; i < RF; ++i) {
            id[i] = r0 + i * 16 + s < t.rows_here ? a.ids[t.row0 + r0 + i * 16 + s] : -1;
            if (static_cast<unsigned>(id[i]) >= static_cast<unsigned>(a.adapters)) id[i] = -1;
        }
        if constexpr (kShift) {
            float most[RF];
#pragma unroll
            for (int i = 0; i < RF; ++i) most[i] = 0.0f;
            for (int k0 = 0; k0 < rank; k0 += 32) {
#pragma unroll
                for (int i = 0; i < RF; ++i) {
                    float v[8];
                    read_h(i, k0, id[i] >= 0, v);
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        const float m = fabsf(v[n]);
                        most[i] = m < __builtin_inff() ? fmaxf(most[i], m) : most[i];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < RF; ++i) {
                most[i]  = fmaxf(most[i], __shfl_xor(most[i], 16));
                most[i]  = fmaxf(most[i], __shfl_xor(most[i], 32));
                shift[i] = __builtin_amdgcn_frexp_expf(most[i]) - 14;
            }
        }
    }
    // Eight values of h, from k0 + 8 (lane >> 4) on, of row 16 i + (lane & 15); zeros where
    // the row is not `wanted`, and past the rank.
    __device__ __forceinline__ void read_h(int i, int k0, bool wanted, float (&v)[8]) const {
        const int lane = threadIdx.x & 63;
        const int k = k0 + 8 * (lane >> 4);
        const float* at = h + (i * 16 + (lane & 15)) * rank16 + k;
        uint4 x{}, y{};
        if (wanted && k < rank16) {
            x = load_piece(at);
            y = load_piece(at + 4);
        }
        __builtin_memcpy(v, &x, 16);
        __builtin_memcpy(v + 4, &y, 16);
    }
    // B_a's rows c0 .. of an adapter, 32 of the rank from k0 on.
    __device__ __forceinline__ void read_b(int adapter, int k0, Operand<T> (&fc)[CF]) const {
        const int k = k0 + 8 * ((threadIdx.x & 63) >> 4);
        const int here = min(width - c0, CF * 16);  // may be below 1
        const T* first = b + (static_cast<long long>(adapter) * width + c0) * rank;
        const unsigned odd = PIECES ? 0u : static_cast<unsigned>(reinterpret_cast<uintptr_t>(first)) & 2u;
        const __amdgpu_buffer_rsrc_t buffer = words_buffer(first, static_cast<long long>(max(here, 0)) * rank);
#pragma unroll
        for (int j = 0; j < CF; ++j) {
            const int c = j * 16 + (threadIdx.x & 15);
            const unsigned at = c < here && k < rank ? static_cast<unsigned>(c * rank + k) * 2u + odd
                                                     : kAbsent;
            const WordPiece v = load_words<!PIECES>(buffer, at);
            fc[j] = __builtin_bit_cast(Operand<T>, PIECES ? v.words : first_of(piece_of(v, at), rank - k));
        }
    }
    // Sums for the rows 16 i .. that `adapter` has (`own`), of both parts of h or the high
    // one alone.  kept: the parts of the rank's first kKept x 32, of every row.
    template <bool LOW>
    __device__ __forceinline__ void multiply(int i, int adapter, bool own, int up,
                                             const Parts<T> (&kept)[kKept], f32x4 (&sum)[CF]) const {
#pragma unroll
        for (int j = 0; j < CF; ++j) sum[j] = f32x4(0.0f);
        for (int k0 = 0; k0 < rank; k0 += 32) {
            Operand<T> fc[CF];
            read_b(adapter, k0, fc);
            Parts<T> fr;
            if (k0 < 32 * kKept) {
                const Parts<T> all = kKept == 1 || k0 == 0 ? kept[0] : kept[kKept - 1];
                const Operand<T> none = __builtin_bit_cast(Operand<T>, uint4{});
                fr = Parts<T>{own ? all.high : none, own ? all.low : none};
            } else {
                float v[8];
                read_h(i, k0, own, v);
                fr = parts_of<T>(v, up);
            }
            if constexpr (LOW) {
#pragma unroll
                for (int j = 0; j < CF; ++j) sum[j] = mfma(fc[j], fr.low, sum[j]);
            }
#pragma unroll
            for (int j = 0; j < CF; ++j) sum[j] = mfma(fc[j], fr.high, sum[j]);
        }
    }
    // sums: the wave's rows 16 i .. in LDS, `pitch` floats a row; mine, up: id[i], shift[i].
    // An infinity in h or B can make the two parts inf - inf or 0 inf where their sum is an
    // infinity: those elements take the high part's sum.
    __device__ __forceinline__ void add(int i, int mine, int up, float* sums, int pitch) const {
        const int lane = threadIdx.x & 63;
        float* at = sums + (lane & 15) * pitch + 4 * (lane >> 4);
        int left_id = mine;
        unsigned long long left = __ballot(left_id >= 0);
        if (left == 0) return;
        Parts<T> kept[kKept];
#pragma unroll
        for (int n = 0; n < kKept; ++n) {
            float v[8];
            read_h(i, 32 * n, mine >= 0, v);
            kept[n] = parts_of<T>(v, up);
        }
        for (; left != 0; left = __ballot(left_id >= 0)) {
            const int adapter = __builtin_amdgcn_readlane(left_id, __builtin_ctzll(left));
            const bool own = mine == adapter;
            f32x4 sum[CF];
            multiply<true>(i, adapter, own, up, kept, sum);
            f32x4 none(0.0f);  // stays 0 while all are finite
#pragma unroll
            for (int j = 0; j < CF; ++j) none = sum[j] * 0.0f + none;
            const bool finite = (none[0] + none[1]) + (none[2] + none[3]) == 0.0f;
            if (__ballot(own && !finite) != 0) {
                f32x4 high[CF];
                multiply<false>(i, adapter, own, up, kept, high);
#pragma unroll
                for (int j = 0; j < CF; ++j)
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        sum[j][n] = fabsf(sum[j][n]) < __builtin_inff() ? sum[j][n] : high[j][n];
                    }
            }
            if (own) {
#pragma unroll
                for (int j = 0; j < CF; ++j) {
                    f32x4* p = reinterpret_cast<f32x4*>(at + 16 * j);
                    f32x4 more = sum[j];
                    if constexpr (kShift) {
#pragma unroll
                        for (int n = 0; n < 4; ++n) more[n] = ldexpf(more[n], up);
                    }
                    *p = *p + more;
                }
            }
            left_id = own ? -1 : left_id;
        }
    }
};

// Eight columns of a row on their way out, c .. of them the first `count` (none: 0).  Gated:
// g and u, which leave as act(g) u and, where they are kept, as they are or packed (four
// lanes a block; all 64 come here).
template <typename T, bool GATED>
__device__ __forceinline__ void finish_row(const TileArgs& a, long long row, int c, int count,
                                           float (&f)[GATED ? 2 : 1][8]) {
    const auto store = [&](void* to, long long at, const float (&v)[8]) {
        if constexpr (std::is_same_v<T, Int8Pair>) store_eight_as(to, a.out_type, at, v, count);
        else store_eight(static_cast<T*>(to) + at, v, count);
    };
    if constexpr (GATED && !std::is_same_v<T, Int8Pair>) {
        if (a.kept_scales != nullptr) {
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                const unsigned scale = pack_scale(quad_max(largest_bits(f[part])));
                if (count <= 0) continue;
                const long long line = 2 * row + part;
                store_bytes(static_cast<signed char*>(a.kept) + line * a.width + c,
                            pack_eight(f[part], scale), count);
                if (c % kPackBlock == 0) {
                    const long long blocks = (a.width + kPackBlock - 1) / kPackBlock;
                    a.kept_scales[line * blocks + c / kPackBlock] = static_cast<unsigned char>(scale);
                }
            }
        } else if (a.kept != nullptr && count > 0) {
#pragma unroll
            for (int part = 0; part < 2; ++part) store(a.kept, (2 * row + part) * a.width + c, f[part]);
        }
    }
    if (count <= 0) return;
    if constexpr (GATED) {
        float h[8];
        gate_values(a.act, f[0], h);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] *= f[1][e];
        store(a.out, row * a.width + c, h);
    } else {
        store(a.out, row * a.width + c, f[0]);
    }
}

// Floats of LDS that a wave's stores take: sixteen rows of its columns, four more
// a row so that rows start 16 bytes apart in the banks.
template <int CF>
constexpr int kStoreFloats = 16 * (CF * 16 + 4);

// Stores a wave's tile, sixteen rows at a time through its own part of LDS (`sums`,
// free in all waves), so that whole row pieces leave in 16-byte stores.
template <typename T, int RF, int CF>
struct StoreTile {
    static constexpr int kPitch = CF * 16 + 4, kLanes = CF * 2, kRows = 64 / kLanes;
    const TileArgs& a;
    const Tile<T>&  t;
    int    r0, c0;
    float* sums;

    template <int I>
    __device__ __forceinline__ void put(const f32x4 (&acc)[CF][RF]) const {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int j = 0; j < CF; ++j) {
            *reinterpret_cast<f32x4*>(sums + (lane & 15) * kPitch + j * 16 + 4 * (lane >> 4)) = acc[j][I];
        }
    }
    // SCALED: lane l < 16 holds what row l's sums are multiplied by.
    template <bool SCALED = false>
    __device__ __forceinline__ void store(int i, float scale = 1.0f) const {
        const int lane = threadIdx.x & 63;
        const int c = c0 + lane % kLanes * 8;
        const int count = min(8, a.width - c);
#pragma unroll
        for (int n = 0; n < 16 / kRows; ++n) {
            const int r = n * kRows + lane / kLanes;
            const float* from = sums + r * kPitch + lane % kLanes * 8;
            float f[8];
            __builtin_memcpy(f, __builtin_assume_aligned(from, 16), 32);
            if constexpr (SCALED) {
                const float by = __shfl(scale, r);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] *= by;
            }
            const uint4 v = piece_from_float<T>(f);
            if (r0 + i * 16 + r < t.rows_here && count > 0) {
                T* p = t.out + static_cast<long long>(r0 + i * 16 + r) * a.width + c;
                if (count == 8) store_piece(p, v);
                else store_part(p, v, count);
            }
        }
    }
};
template <typename T, int RF, int CF, bool SCALED>
__device__ __forceinline__ void store_tile(const TileArgs& a, const Tile<T>& t, int r0, int c0,
                                           const f32x4 (&acc)[CF][RF], float* sums) {
    const StoreTile<T, RF, CF> tile{a, t, r0, c0, sums};
    float scale[RF];  // all rows' loads before the first store
    if constexpr (SCALED) {
#pragma unroll
        for (int i = 0; i < RF; ++i) {
            const int row = r0 + i * 16 + (threadIdx.x & 15);
            scale[i] = a.group_scales != nullptr ? a.group_scales[t.group]
                       : row < t.rows_here ? a.row_scales[t.row0 + row] : 0.0f;
        }
    }
    unrolled(std::make_integer_sequence<int, RF>{}, [&](auto at) {
        if (r0 + at.value * 16 < t.rows_here) {
            tile.template put<at.value>(acc);
            if constexpr (SCALED) tile.template store<true>(at.value, scale[at.value]);
            else tile.store(at.value);
        }
    });
}

// The gated and the scaled stores of a wave's tile, B sixteens of rows at a time through its
// own part of LDS (one at a time, each waits for its own way through LDS and for its own
// functions: 20800 rows x 2 x 3776 x 128 in 256 x 256 tiles 208 us, 136 with four).  Gated,
// the first half of a row's sums are the gates and the second half what they multiply, of
// the same kCols columns; a lane takes eight columns of both, four lanes a block of 32 for
// packing.
template <typename T, int CF, bool GATED, int B>
struct FinishTile {
    static constexpr bool kScaled = std::is_same_v<T, Int8Pair>;
    static constexpr int  kPitch = CF * 16 + 4, kCols = GATED ? CF * 8 : CF * 16;
    static constexpr int  kLanes = kCols / 8, kRows = 64 / kLanes;
    static constexpr int  kParts = GATED ? 2 : 1;
    const TileArgs& a;
    const Tile<T>&  t;
    int    c, count;  // the lane's first column, and how many of its eight there are
    float* sums;
    float  scale[kScaled ? kParts : 1][8];  // of the lane's columns

    __device__ __forceinline__ FinishTile(const TileArgs& args, const Tile<T>& tile, int col, float* lds)
        : a(args), t(tile), c(col + (threadIdx.x & 63) % kLanes * 8), count(min(8, a.width - c)),
          sums(lds) {
        if constexpr (kScaled) {
            const float* from = a.col_scales + static_cast<long long>(t.group) * kParts * a.width;
#pragma unroll
            for (int part = 0; part < kParts; ++part)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    scale[part][e] = e < count ? from[static_cast<long long>(part) * a.width + c + e] : 0.0f;
                }
        }
    }
    // A sixteen's sums into place k.
    __device__ __forceinline__ void put(int k, int j, Sums<T> x) const {
        const int lane = threadIdx.x & 63;
        f32x4 v;
#pragma unroll
        for (int n = 0; n < 4; ++n) v[n] = static_cast<float>(x[n]);
        *reinterpret_cast<f32x4*>(sums + (k * 16 + (lane & 15)) * kPitch + j * 16 + 4 * (lane >> 4)) = v;
    }
    // Rows row0 .. of the tile, from the first place on.
    __device__ __forceinline__ void store(int row0) const {
        const int lane = threadIdx.x & 63;
#pragma unroll 2
        for (int n = 0; n < B * 16 / kRows; ++n) {
            const int r = n * kRows + lane / kLanes, row = row0 + r;
            const float* from = sums + r * kPitch + lane % kLanes * 8;
            float f[kParts][8];
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
                __builtin_memcpy(f[part], __builtin_assume_aligned(from + part * kCols, 16), 32);
            }
            if constexpr (kScaled) {
                const float s = row < t.rows_here ? a.row_scales[t.row0 + row] : 0.0f;
#pragma unroll
                for (int part = 0; part < kParts; ++part)
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[part][e] = f[part][e] * scale[part][e] * s;
            }
            finish_row<T, GATED>(a, t.row0 + row, c, row < t.rows_here ? count : 0, f);
        }
    }
};
template <typename T, int RF, int CF, bool GATED, int B>
__device__ __forceinline__ void finish_tile(const TileArgs& a, const Tile<T>& t, int r0, int c0,
                                            const Sums<T> (&acc)[CF][RF], float* sums) {
    const FinishTile<T, CF, GATED, B> tile(a, t, c0, sums);
    unrolled(std::make_integer_sequence<int, RF / B>{}, [&](auto at) {
        constexpr int first = at.value * B;
        if (r0 + first * 16 < t.rows_here) {
            unrolled(std::make_integer_sequence<int, B * CF>{}, [&](auto m) {
                tile.put(m.value / CF, m.value % CF, acc[m.value % CF][first + m.value / CF]);
            });
            tile.store(r0 + first * 16);
        }
    });
}

// How 128 rows (or columns) of an operand's staged tile reach LDS in 16-byte
// pieces by buffer loads of 256 threads: the places of Operands<T, 128, ...>.
// Rows n = 64 p + r of the slot are the operand's rows GAP p + r.
template <typename T, bool MAJOR, int GAP>
struct Slot {
    static constexpr int kPieces = 4;
    static constexpr int kBytes  = 128 * kStep * 2;
    unsigned at[kPieces];  // byte offset of the piece; past every buffer's end for no such row
    int      index;        // its first contraction step, less 16 i for MAJOR

    __device__ __forceinline__ void place(int ld, int first, int bound) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int p = i * 256 + threadIdx.x;
            int k, n;  // contraction step, row of the slot
            if constexpr (MAJOR) {
                k = p / 16;
                const int f = (k & 3) | ((k >> 3) & 1) << 2;
                n = ((p % 16) ^ (f << 1)) * 8;
            } else {
                n = p / 8;
                k = ((p % 8) ^ (n & 7)) * 8;
            }
            const int row = first + (n / 64) * GAP + n % 64;
            const int element = MAJOR ? k * ld + row : row * ld + k;
            at[i] = row < bound ? static_cast<unsigned>(element) * 2u : kAbsent;
            if (i == 0) index = k;
        }
    }
    // Where piece I of a tile with `left` contraction steps left lies.
    template <int I>
    __device__ __forceinline__ unsigned offset(int left) const {
        return index + (MAJOR ? 16 * I : 0) < left ? at[I] : kAbsent;
    }
};

// Stores a wave's tile with its rows' adapters added.
template <typename T, int RF, int CF>
__device__ __forceinline__ void store_adapted(const TileArgs& a, const Tile<T>& t, int r0, int c0,
                                              const f32x4 (&acc)[CF][RF], float* sums) {
    auto store = [&](auto pieces) {
        const Adapters<T, RF, CF, pieces.value> ad(a, t, r0, c0);
        const StoreTile<T, RF, CF> tile{a, t, r0, c0, sums};
        // one body for all sixteens of rows: they are gone through once, and as many bodies
        // would come from memory first (8192 rows x 4096 x 4096, rank 64, an adapter a run of
        // rows: fp16 254 us, 262 so; a different one a row 668 both, 748 with the parts made
        // again for each)
#pragma unroll 1
        for (int i = 0; i < RF && r0 + i * 16 < t.rows_here; ++i) {
            int mine = -1, up = 0;
            unrolled(std::make_integer_sequence<int, RF>{}, [&](auto at) {
                if (at.value == i) {
                    tile.template put<at.value>(acc);
                    mine = ad.id[at.value];
                    if constexpr (ad.kShift) up = ad.shift[at.value];
                }
            });
            ad.add(i, mine, up, sums, tile.kPitch);
            tile.store(i);
        }
    };
    if (a.b_pieces) store(std::true_type{});
    else store(std::false_type{});
}

// The same where the sums are scaled or gated: whole waves go through the rows.
template <int COLS, typename T, bool GATED>
__device__ __forceinline__ void finish_zeros(const TileArgs& a, const Tile<T>& t) {
    const int c = t.c0 + threadIdx.x % (COLS / 8) * 8;
    const int step = blockDim.x / (COLS / 8);
    for (int r = threadIdx.x / (COLS / 8); r - static_cast<int>(threadIdx.x / (COLS / 8)) < t.rows_here;
         r += step) {
        float f[GATED ? 2 : 1][8] = {};
        finish_row<T, GATED>(a, t.row0 + r, c, r < t.rows_here ? min(8, a.width - c) : 0, f);
    }
}
// Zeros where nothing is summed: rows in no group, the gradient of an empty one.
template <int BC, typename T>
__device__ __forceinline__ void zero_tile(const TileArgs& a, const Tile<T>& t) {
    const int c = t.c0 + threadIdx.x % (BC / 8) * 8;
    const int count = min(8, a.width - c);
    if (count <= 0) return;
    for (int r = threadIdx.x / (BC / 8); r < t.rows_here; r += blockDim.x / (BC / 8)) {
        T* p = t.out + static_cast<long long>(r) * a.width + c;
        if (count == 8) store_piece(p, uint4{});
        else store_part(p, uint4{}, count);
    }
}

// How operands lie in memory for buffer-to-LDS loads: rows of whole 16-byte pieces, of whole
// words, or of 16-bit elements that may begin between two words.
enum class Lie { Pieces, Words, Odd };

// A buffer from `at` (down to its word) on; past `end` (up to its word) there are zeros.
// Pieces need no end: each is there as a whole or absent.
template <Lie L>
__device__ __forceinline__ u32x4 operand_words(const void* at, const void* end) {
    if constexpr (L == Lie::Pieces) return buffer_words(at, 0, 0x7fffffff);
    const uintptr_t from = reinterpret_cast<uintptr_t>(at) & ~uintptr_t{3};
    const long long left = static_cast<long long>((reinterpret_cast<uintptr_t>(end) + 3) & ~uintptr_t{3}) -
                           static_cast<long long>(from);
    // compared by halves: the scalar unit compares no 64 bits
    const int high = static_cast<int>(left >> 32);
    const unsigned low = static_cast<unsigned>(left), most = 0x7ffffffcu;
    const unsigned records = high < 0 ? 0u : high > 0 || low > most ? most : low;
    return buffer_words(reinterpret_cast<const void*>(from), 0, static_cast<int>(records));
}

// Whether a tile's sums leave through store_tile (or with adapters).
template <typename T, Ends E>
constexpr bool kPlainEnds = E != Ends::Gated && !std::is_same_v<T, Int8Pair>;

// Floats of LDS that a wave's end takes.  B: sixteens of rows that gated and scaled sums leave in.
template <typename T, int CF, Ends E, int B>
constexpr int kLeaveFloats = kStoreFloats<CF> * (kPlainEnds<T, E> ? 1 : B);

template <typename T, int RF, int CF, Ends E, int B>
__device__ __forceinline__ void leave(const TileArgs& a, const Tile<T>& t, int r0, int c0,
                                      const Sums<T> (&acc)[CF][RF], char* lds, int wave) {
    float* sums = reinterpret_cast<float*>(lds) + wave * kLeaveFloats<T, CF, E, B>;
    if constexpr (!kPlainEnds<T, E>) {
        finish_tile<T, RF, CF, E == Ends::Gated, B>(a, t, r0, c0, acc, sums);
    } else if constexpr (E == Ends::Adapters) {
        store_adapted<T, RF, CF>(a, t, r0, c0, acc, sums);
    } else {
        store_tile<T, RF, CF, E == Ends::Scaled>(a, t, r0, c0, acc, sums);
    }
}

// GRAD false: a product (rows operand [s][k], columns operand W as COLS_MAJOR
// says).  GRAD true: a weight gradient (both operands lie along s).
// E: how the sums leave.  Gated tiles hold half as many of the output's columns, the gates'
// sums and the others' next to each other in a wave, which needs both.
//
// The 128 x 128 tile of medium products, and of any sizes and alignment: four waves
// take a quarter each, two buffers of 64 steps.  The operands' rows of whole 16-byte
// pieces or words go straight into LDS (words cut there as in tile_product_wide).  Odd:
// others go through registers, as the words around each piece, from buffers that end with the operand:
// straight code with eight or sixteen loads under way.  (With a branch a piece for those
// at an edge the compiler waited for each load: 8 groups of 4000 x 4098 over 16384 rows
// 930 us, 810 so; their weights' gradient 1280, 790.  Two workgroups a CU need the
// registers bounded: 1390 with one.)
template <typename T, bool GRAD, bool COLS_MAJOR, Ends E, Lie L>
__global__ __launch_bounds__(256, L == Lie::Odd ? 2 : 1) void tile_product(TileArgs a) {
    constexpr bool GATED = E == Ends::Gated;
    constexpr int BR = 128, BC = 128, WC = 2, RF = 4, CF = 4, OUT = GATED ? BC / 2 : BC;
    using Rows = Operands<T, BR, GRAD, 256>;
    using Cols = Operands<T, BC, GRAD || COLS_MAJOR, 256, GATED ? 2 : 1>;
    __shared__ __attribute__((aligned(16))) T s_tiles[2 * (BR + BC) * kStep];
    auto rows_at = [&](int it) { return s_tiles + (it & 1) * BR * kStep; };
    auto cols_at = [&](int it) { return s_tiles + (2 * BR + (it & 1) * BC) * kStep; };

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave / WC, wc = wave % WC;
    Tile<T> t;
    if (!take_tile<T, BR, OUT, GRAD, COLS_MAJOR, GATED>(a, t)) return;

    Sums<T> acc[CF][RF];
#pragma unroll
    for (int j = 0; j < CF; ++j)
#pragma unroll
        for (int i = 0; i < RF; ++i) acc[j][i] = Sums<T>(0);

    const int r0 = wr * RF * 16, c0 = t.c0 + wc * (OUT / WC);
    const int tiles = (t.depth + kStep - 1) / kStep;
    if constexpr (!kPlainEnds<T, E>) {
        if (tiles == 0) return finish_zeros<OUT, T, GATED>(a, t);
    }
    // the staged column that a wave's 16 columns j begin at
    auto column = [&](int j) {
        return GATED ? j / (CF / 2) * (BC / 2) + (wc * (CF / 2) + j % (CF / 2)) * 16 : (wc * CF + j) * 16;
    };
    auto multiply = [&](int it) {
        const T* lr = rows_at(it);
        const T* lc = cols_at(it);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            Operand<T> fr[RF], fc[CF];
#pragma unroll
            for (int i = 0; i < RF; ++i) fr[i] = Rows::read(lr, (wr * RF + i) * 16, half);
#pragma unroll
            for (int j = 0; j < CF; ++j) fc[j] = Cols::read(lc, column(j), half);
#pragma unroll
            for (int j = 0; j < CF; ++j)
#pragma unroll
                for (int i = 0; i < RF; ++i) acc[j][i] = mfma(fc[j], fr[i], acc[j][i]);
        }
    };
    if constexpr (L != Lie::Odd) {
        Slot<T, GRAD, 64> pr;
        Slot<T, GRAD || COLS_MAJOR, GATED ? 0 : 64> pc;
        pr.place(t.ld_rows, 0, t.rows_here);
        pc.place(t.ld_cols, 0, a.width - t.c0);
        auto load = [&](int it) {
            const u32x4 br = operand_words<L>(t.rows + it * t.step_rows, a.rows_end);
            const u32x4 bc = operand_words<L>(t.cols + it * t.step_cols, a.cols_end);
            const u32x4 bs = GATED ? operand_words<L>(t.second + it * t.step_cols, a.cols_end) : bc;
            const unsigned lr = lds_address(rows_at(it)) + wave * 1024;
            const unsigned lc = lds_address(cols_at(it)) + wave * 1024;
            const int left = t.depth - it * kStep;
            unrolled(std::make_integer_sequence<int, 4>{}, [&](auto i) {
                lds_dma_raw_to<i.value * 4096>(lr);
                asm volatile("s_nop 0");
                lds_dma_raw_x4(br, pr.template offset<i.value>(left));
                lds_dma_raw_to<i.value * 4096>(lc);
                asm volatile("s_nop 0");
                lds_dma_raw_x4(i.value < 2 ? bc : bs, pc.template offset<i.value>(left));
            });
        };
        if (tiles > 0) load(0);
        for (int it = 0; it < tiles; ++it) {
            // every wave's pieces are there, and the other buffer's readers are done
            wait_vmcnt<0>();
            lds_barrier();
            if (L == Lie::Words && !GRAD && it + 1 == tiles && t.depth % 8 != 0) {
                const int last = t.depth - it * kStep, n = threadIdx.x & 127;
                if (threadIdx.x < 128 || !COLS_MAJOR) {
                    T* row = (threadIdx.x < 128 ? rows_at(it) : cols_at(it)) + n * kStep;
                    uint4* piece = reinterpret_cast<uint4*>(row) + ((last / 8) ^ (n & 7));
                    *piece = first_of(*piece, last % 8);
                }
                lds_barrier();
            }
            if (it + 1 < tiles) load(it + 1);
            multiply(it);
        }
    } else {
        Rows pr;
        Cols pc;
        pr.place(t.rows, t.ld_rows, t.rows_here);
        pc.place(t.cols, t.ld_cols, a.width - t.c0, GATED ? t.second : nullptr);
        WordPiece vr[Rows::kPieces], vc[Cols::kPieces];
        auto run = [&](auto odd) {
            auto load = [&](int it) {
                const int left = t.depth - it * kStep;
                pr.template load<odd.value>(t.rows + it * t.step_rows, left, vr);
                pc.template load<odd.value>(t.cols + it * t.step_cols, left, vc,
                                                GATED ? t.second + it * t.step_cols : nullptr);
            };
            auto store = [&](int it) {
                const int left = t.depth - it * kStep;
                pr.template store<odd.value>(rows_at(it), left, vr);
                pc.template store<odd.value>(cols_at(it), left, vc);
            };
            load(0);
            store(0);
            for (int it = 0; it < tiles; ++it) {
                // the tile is written, and the other buffer's readers are done
                __syncthreads();
                if (it + 1 < tiles) load(it + 1);
                multiply(it);
                if (it + 1 < tiles) store(it + 1);
            }
        };
        const uintptr_t ends = reinterpret_cast<uintptr_t>(t.rows) | reinterpret_cast<uintptr_t>(t.cols) |
                               (GATED ? reinterpret_cast<uintptr_t>(t.second) : 0) |
                               static_cast<uintptr_t>(t.ld_rows | t.ld_cols) * 2;
        if (tiles == 0) {
        } else if ((ends & 2) != 0) {
            run(std::true_type{});
        } else {
            run(std::false_type{});
        }
    }
    lds_barrier();  // the operands' LDS is free
    static_assert(WC * 2 * kLeaveFloats<T, CF, E, 2> * sizeof(float) <= sizeof(s_tiles), "LDS of the ends");
    leave<T, RF, CF, E, 2>(a, t, r0, c0, acc, reinterpret_cast<char*>(s_tiles), wave);
}

// The 64 x 64 tile of products with few tiles and a long contraction: sixteen waves in
// four groups share the contraction, each with its own two buffers, and add up in a fixed
// order.  Any sizes and alignment, as the words around each piece.  Bound by a load's way
// through registers into LDS, about 1 us a turn of 256 steps.  128 rows x 64 x 5120, W
// [k][c], two such tiles or one of 128 x 128: 25 us, 46 with the latter; 1024 x 1024 x
// 4096 24, 43; 823 x 768 x 6787 with adapters 70, 145; a gradient of 256 x 256 from 32768
// rows 136, 287.
template <typename T, bool GRAD, bool COLS_MAJOR, Ends E>
__global__ __launch_bounds__(1024) void tile_product_shared(TileArgs a) {
    static_assert(kPlainEnds<T, E>);
    constexpr int BR = 64, BC = 64, WC = 2, RF = 2, CF = 2, GROUPS = 4;
    using Rows = Operands<T, BR, GRAD, 256>;
    using Cols = Operands<T, BC, GRAD || COLS_MAJOR, 256>;
    extern __shared__ __attribute__((aligned(16))) char s_tiles[];
    const int group = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const int wave  = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
    T* const own = reinterpret_cast<T*>(s_tiles) + group * 2 * (BR + BC) * kStep;
    auto rows_at = [&](int it) { return own + (it & 1) * (BR + BC) * kStep; };
    auto cols_at = [&](int it) { return rows_at(it) + BR * kStep; };
    const int wr = wave / WC, wc = wave % WC;
    Tile<T> t;
    if (!take_tile<T, BR, BC, GRAD, COLS_MAJOR>(a, t)) return;

    Sums<T> acc[CF][RF];
#pragma unroll
    for (int j = 0; j < CF; ++j)
#pragma unroll
        for (int i = 0; i < RF; ++i) acc[j][i] = Sums<T>(0);
    const int r0 = wr * RF * 16, c0 = t.c0 + wc * (BC / WC);
    // all groups go through as many turns: past the end there are zeros
    const int turns = (t.depth + GROUPS * kStep - 1) / (GROUPS * kStep);
    Rows pr;
    Cols pc;
    pr.place(t.rows, t.ld_rows, t.rows_here);
    pc.place(t.cols, t.ld_cols, a.width - t.c0);
    WordPiece vr[Rows::kPieces], vc[Cols::kPieces];
    auto run = [&](auto odd) {
        auto load = [&](int it) {
            const int n = it * GROUPS + group, left = t.depth - n * kStep;
            pr.template load<odd.value>(t.rows + n * t.step_rows, left, vr);
            pc.template load<odd.value>(t.cols + n * t.step_cols, left, vc);
        };
        auto store = [&](int it) {
            const int left = t.depth - (it * GROUPS + group) * kStep;
            pr.template store<odd.value>(rows_at(it), left, vr);
            pc.template store<odd.value>(cols_at(it), left, vc);
        };
        load(0);
        store(0);
        for (int it = 0; it < turns; ++it) {
            __syncthreads();
            if (it + 1 < turns) load(it + 1);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                Operand<T> fr[RF], fc[CF];
#pragma unroll
                for (int i = 0; i < RF; ++i) fr[i] = Rows::read(rows_at(it), (wr * RF + i) * 16, half);
#pragma unroll
                for (int j = 0; j < CF; ++j) fc[j] = Cols::read(cols_at(it), (wc * CF + j) * 16, half);
#pragma unroll
                for (int j = 0; j < CF; ++j)
#pragma unroll
                    for (int i = 0; i < RF; ++i) acc[j][i] = mfma(fc[j], fr[i], acc[j][i]);
            }
            if (it + 1 < turns) store(it + 1);
        }
    };
    const uintptr_t ends = reinterpret_cast<uintptr_t>(t.rows) | reinterpret_cast<uintptr_t>(t.cols) |
                           static_cast<uintptr_t>(t.ld_rows | t.ld_cols) * 2;
    if (turns > 0) {
        if ((ends & 2) != 0) run(std::true_type{});
        else run(std::false_type{});
    }
    __syncthreads();  // the operands' LDS is free
    Sums<T>(*parts)[4][CF][RF][64] = reinterpret_cast<Sums<T>(*)[4][CF][RF][64]>(s_tiles);
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < CF; ++j)
#pragma unroll
        for (int i = 0; i < RF; ++i) parts[group][wave][j][i][lane] = acc[j][i];
    __syncthreads();
    if (group != 0) return;
#pragma unroll
    for (int j = 0; j < CF; ++j)
#pragma unroll
        for (int i = 0; i < RF; ++i) {
            for (int g = 1; g < GROUPS; ++g) acc[j][i] = acc[j][i] + parts[g][wave][j][i][lane];
        }
    // behind the shares: the other waves may still read theirs
    leave<T, RF, CF, E, 1>(a, t, r0, c0, acc, s_tiles + sizeof(*parts) * GROUPS, wave);
}

// The 256 x 256 tile of large products, for operands whose rows are whole 16-byte
// pieces or words.  Four waves, one a SIMD, take a quarter of 128 x 128 each; 64 steps of
// the contraction are a tile of four slots of 16 KB in LDS: columns 0-127 (C0) and
// 128-255 (C1), the first 64 rows of either pair of waves (L) and the last 64 (H).
// Ten slots form a ring, filled by buffer-to-LDS loads in the order C0 C1 L H.
//
// A tile is multiplied in four parts: L with the first 32 steps and the last 32,
// then H (the columns' operands stay in registers).  Behind a part's products the
// wave issues the next part's operand reads and one slot's loads.  C0, C1 and L are
// read by the end of part 0, H by the end of part 2; a barrier behind each of these
// frees their slots.  So slot n is loaded seven parts before it is read, about two
// tiles ahead: with two buffers of a tile (a quarter of that ahead) waves stood
// still for a sixth of the time, loads that miss the L2 being waited for.
//   Before the barriers each wave waits for its own loads: behind part 2 all but
//   the five youngest slots (the next tile's C0, C1, L are there), behind part 0
//   all but six (this tile's H is there), and for its operand reads.
//   Past the contraction's end loads write zeros, so the counts always hold.
//   Words: the last piece of a row may hold the next row's first elements, which are cut off
//     in LDS before its slot is read (contraction along rows; other operands only have them
//     in columns past the tile's).
//
// 8 groups of 8192 x 4096 over 16384 rows: 887 us a call, 1240 TFLOP/s (the kernel alone
// 869 at best); in one group 783 us at best, 1400, and 808 on average.  The matrix cores
// are busy for 73% of the time, and at that the clock falls to 1.4 - 1.65 GHz (data of
// zeros takes a sixth less time).  That is no limit of the card: a library product of the
// one group keeps them at 89% and takes 740 at best, 789 on average.  What is left lies in
// the two barriers a tile, with their waits for loads, and in the 6 us that a tile costs
// beside its 1.55 us for 64 steps: beginning, first loads and stores.
template <typename T, bool GRAD, bool COLS_MAJOR, Ends E, Lie L = Lie::Pieces>
__global__ __launch_bounds__(256, 1) void tile_product_wide(TileArgs a) {
    static_assert(L != Lie::Odd, "rows of whole words");
    constexpr bool GATED = E == Ends::Gated;
    constexpr int BR = 256, BC = 256, RF = 8, CF = 8, OUT = GATED ? BC / 2 : BC;
    using RowSlot = Slot<T, GRAD, 128>;
    using ColSlot = Slot<T, GRAD || COLS_MAJOR, GATED ? 0 : 64>;
    using Rows = Operands<T, 128, GRAD, 256>;
    using Cols = Operands<T, 128, GRAD || COLS_MAJOR, 256>;
    extern __shared__ __attribute__((aligned(16))) char s_tiles[];
    constexpr int kSlot = 128 * kStep;  // elements

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave >> 1, wc = wave & 1;
    Tile<T> t;
    if (!take_tile<T, BR, OUT, GRAD, COLS_MAJOR, GATED>(a, t)) return;

    Sums<T> acc[CF][RF];
    const int r0 = wr * RF * 16, c0 = t.c0 + wc * (OUT / 2);
    const int tiles = (t.depth + kStep - 1) / kStep;
    if (tiles == 0) {
        if constexpr (kPlainEnds<T, E>) return zero_tile<BC>(a, t);
        else return finish_zeros<OUT, T, GATED>(a, t);
    }
    {
        ColSlot cols0, cols1;
        RowSlot low, high;
        cols0.place(t.ld_cols, 0, a.width - t.c0);
        cols1.place(t.ld_cols, OUT / 2, a.width - t.c0);
        low.place(t.ld_rows, 0, t.rows_here);
        high.place(t.ld_rows, 64, t.rows_here);
        T* const lds = reinterpret_cast<T*>(s_tiles);
        const unsigned lds0 = lds_address(s_tiles) + wave * 1024;
        auto place_of = [&](int slot) { return lds0 + slot * ColSlot::kBytes; };
        // The tile that is being loaded, as buffers that begin at it, and the
        // contraction steps left there.
        u32x4 rows = operand_words<L>(t.rows, a.rows_end);
        u32x4 cols = operand_words<L>(t.cols, a.cols_end);
        u32x4 second = GATED ? operand_words<L>(t.second, a.cols_end) : cols;
        int left = t.depth;
        long long steps = 0;
        auto step = [](u32x4& buffer, long long bytes) {
            const unsigned long long at =
                (static_cast<unsigned long long>(buffer[1]) << 32 | buffer[0]) + bytes;
            buffer[0] = static_cast<unsigned>(at);
            buffer[1] = static_cast<unsigned>(at >> 32);
        };
        auto advance = [&] {
            left -= kStep;
            if constexpr (L == Lie::Words) {
                ++steps;
                rows = operand_words<L>(t.rows + steps * t.step_rows, a.rows_end);
                cols = operand_words<L>(t.cols + steps * t.step_cols, a.cols_end);
                if constexpr (GATED) second = operand_words<L>(t.second + steps * t.step_cols, a.cols_end);
                return;
            }
            step(rows, t.step_rows * 2);
            step(cols, t.step_cols * 2);
            if constexpr (GATED) step(second, t.step_cols * 2);
        };
        // Cuts the rows of a tile's slots off at their end: the columns' (two threads a pair of
        // slots) or one of rows.
        const int last = t.depth - (tiles - 1) * kStep;
        const bool partial = L == Lie::Words && !GRAD && last % 8 != 0;
        auto cut = [&](int slot) {
            const int n = threadIdx.x & 127;
            uint4* piece = reinterpret_cast<uint4*>(s_tiles + slot * ColSlot::kBytes + n * kStep * 2 +
                                                    ((last / 8) ^ (n & 7)) * 16);
            *piece = first_of(*piece, last % 8);
        };
        auto cut_cols = [&](int slot0, int slot1, int low_slot) {
            if constexpr (!COLS_MAJOR) cut(threadIdx.x < 128 ? slot0 : slot1);
            if (threadIdx.x < 128) cut(low_slot);
            lds_barrier();
        };
        // what load i of a slot of columns is from
        auto half_of = [&](auto i, const u32x4& from) -> const u32x4& {
            return GATED && i.value >= 2 && &from == &cols ? second : from;
        };
        auto load_slot = [&](const auto& slot, const u32x4& from, unsigned to) {
            unrolled(std::make_integer_sequence<int, 4>{}, [&](auto i) {
                lds_dma_raw_to<i.value * 4096>(to);
                asm volatile("s_nop 0");
                lds_dma_raw_x4(half_of(i, from), slot.template offset<i.value>(left));
            });
        };

        Operand<T> fr[2][RF / 2], fc[2][CF];
        auto read_row = [&](int slot, int half, int i) {
            fr[half][i] = Rows::read(lds + slot * kSlot, wr * 64 + i * 16, half);
        };
        auto read_col = [&](int slot, int half, int j) {
            fc[half][j] = Cols::read(lds + slot * kSlot, j * 16, half);
        };
        // One part's products; behind product m, read(m) and a step of one of the four
        // loads of `slot` into place `to`: never more than two of them, which the
        // matrix cores' own time covers.
        constexpr int kProducts = CF * RF / 2;
        auto multiply = [&](int half, int second, const auto& slot, const u32x4& from, unsigned to,
                            auto read) {
            unsigned offset = 0;
            __builtin_amdgcn_sched_barrier(0);
            unrolled(std::make_integer_sequence<int, kProducts>{}, [&](auto m) {
                constexpr int j = m.value / (RF / 2), i = m.value % (RF / 2);
                mfma_in_place(acc[j][second * (RF / 2) + i], fc[half][j], fr[half][i]);
                read(m);
                if constexpr (m.value % 8 == 2) offset = slot.template offset<m.value / 8>(left);
                if constexpr (m.value % 8 == 4) lds_dma_raw_to<m.value / 8 * 4096>(to);
                if constexpr (m.value % 8 == 6) {
                    lds_dma_raw_x4(half_of(std::integral_constant<int, m.value / 8>{}, from), offset);
                }
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        load_slot(cols0, cols, place_of(0));
        load_slot(cols1, cols, place_of(1));
        load_slot(low, rows, place_of(2));
        load_slot(high, rows, place_of(3));
        advance();
        load_slot(cols0, cols, place_of(4));
        load_slot(cols1, cols, place_of(5));
        load_slot(low, rows, place_of(6));
        load_slot(high, rows, place_of(7));
        advance();
        load_slot(cols0, cols, place_of(8));
        // the sums begin at 0 while the loads are under way
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < CF; ++j)
#pragma unroll
            for (int i = 0; i < RF; ++i) {
                acc[j][i] = Sums<T>(0);
                asm volatile("" : "+a"(acc[j][i]));
            }
        wait_vmcnt<24>();  // slots 0, 1, 2
        lds_barrier();
        if (partial && tiles == 1) cut_cols(0, 1, 2);
#pragma unroll
        for (int i = 0; i < RF / 2; ++i) read_row(2, 0, i);
#pragma unroll
        for (int j = 0; j < CF; ++j) read_col(wc, 0, j);

        int slot = 0;  // of this tile's C0
        auto later = [&](int n) { return slot + n < 10 ? slot + n : slot + n - 10; };
        for (int it = 0; it < tiles; ++it) {
            multiply(0, 0, cols1, cols, place_of(later(9)), [&](auto m) {
                if constexpr (m.value < 8) read_col(later(wc), 1, m.value);
                else if constexpr (m.value < 12) read_row(later(2), 1, m.value - 8);
            });
            wait_vmcnt<24>();
            lds_barrier();
            if (partial && it + 1 == tiles) {
                if (threadIdx.x < 128) cut(later(3));
                lds_barrier();
            }
            multiply(1, 0, low, rows, place_of(slot), [&](auto m) {
                if constexpr (m.value < 4) read_row(later(3), 0, m.value);
            });
            multiply(0, 1, high, rows, place_of(later(1)), [&](auto m) {
                if constexpr (m.value < 4) read_row(later(3), 1, m.value);
            });
            wait_vmcnt<20>();
            lds_barrier();
            if (partial && it + 2 == tiles) cut_cols(later(4), later(5), later(6));
            advance();
            multiply(1, 1, cols0, cols, place_of(later(2)), [&](auto m) {
                if constexpr (m.value < 4) read_row(later(6), 0, m.value);
                else if constexpr (m.value < 12) read_col(later(4 + wc), 0, m.value - 4);
            });
            slot = later(4);
        }
        settle_sums(acc);
        wait_vmcnt<0>();
        lds_barrier();  // the ring is free
    }
    static_assert(4 * kLeaveFloats<T, CF, E, 4> * sizeof(float) <= kRingLds, "LDS of the ends");
    leave<T, RF, CF, E, 4>(a, t, r0, c0, acc, s_tiles, wave);
}

// The tile of 32 RF x 128 of products that the 256 x 256 tiles are too few of, and of rows
// that are no whole pieces: four waves of 16 RF x 64 over a ring of S stages of 64 steps,
// filled by buffer-to-LDS loads S stages ahead, so that reading weights from memory keeps
// up where a CU has one tile.  A stage is multiplied in two halves; a wave reads the next
// half's operands from LDS before it multiplies one.  One barrier a stage, in its middle:
// behind it the stage's slot is free, as all waves hold its second half in registers.
//   Past the contraction's end loads write zeros, so the counts of loads always hold.
//   Words: the last piece of a row may hold the next row's first elements, which are cut
//     off in LDS before its stage is read (contraction along rows; other operands only have
//     them in columns past the tile's).
//   Odd: rows are staged from the word of their first element on, and shifted by one
//     element as they are read, with the word behind a piece, which for a row's last piece
//     of a stage lies in the next stage.
template <typename T, bool GRAD, bool COLS_MAJOR, Ends E, Lie L, int RF>
__global__ __launch_bounds__(256, 1) void tile_product_ring(TileArgs a) {
    constexpr bool GATED = E == Ends::Gated, ODD = L == Lie::Odd;
    constexpr int BR = 32 * RF, BC = 128, WC = 2, CF = 4, OUT = GATED ? BC / 2 : BC;
    constexpr int kRowLoads = BR / 32, kLoads = kRowLoads + 4, kRowBytes = BR * kStep * 2;
    constexpr int kStage = kRowBytes + BC * kStep * 2, S = kRingLds / kStage;
    constexpr int kAhead = ODD ? 3 : 2;  // stages that have to be there before one is read, and one
    static_assert(!ODD || (!GRAD && !COLS_MAJOR), "rows along the contraction are shifted");
    static_assert(!GRAD || RF == 4, "slots of 128 rows");
    using Rows = Operands<T, 128, GRAD, 256>;
    using Cols = Operands<T, 128, GRAD || COLS_MAJOR, 256>;
    extern __shared__ __attribute__((aligned(16))) char s_tiles[];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave / WC, wc = wave % WC;
    const int lane = threadIdx.x & 63, q = lane >> 4, s = lane & 15;
    Tile<T> t;
    if (!take_tile<T, BR, OUT, GRAD, COLS_MAJOR, GATED>(a, t)) return;

    Sums<T> acc[CF][RF];
#pragma unroll
    for (int j = 0; j < CF; ++j)
#pragma unroll
        for (int i = 0; i < RF; ++i) {
            acc[j][i] = Sums<T>(0);
            asm volatile("" : "+a"(acc[j][i]));
        }
    const int r0 = wr * RF * 16, c0 = t.c0 + wc * (OUT / WC);
    const int stages = (t.depth + kStep - 1) / kStep;
    if constexpr (!kPlainEnds<T, E>) {
        if (stages == 0) return finish_zeros<OUT, T, GATED>(a, t);
    }
    auto column = [&](int j) {
        return GATED ? j / (CF / 2) * (BC / 2) + (wc * (CF / 2) + j % (CF / 2)) * 16 : (wc * CF + j) * 16;
    };
    if (stages > 0) {
        Slot<T, GRAD, 64> pr;
        Slot<T, GRAD || COLS_MAJOR, GATED ? 0 : 64> pc;
        pr.place(t.ld_rows, 0, t.rows_here);
        pc.place(t.ld_cols, 0, a.width - t.c0);
        // Odd: whether an operand begins between two words, and the shift of a lane's row
        unsigned odd_rows = 0, odd_cols = 0, odd_second = 0;
        if constexpr (ODD) {
            auto odd = [](const T* p) { return static_cast<unsigned>(reinterpret_cast<uintptr_t>(p)) & 2u; };
            odd_rows = odd(t.rows);
            odd_cols = odd(t.cols);
            odd_second = GATED ? odd(t.second) : odd_cols;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (pr.at[i] != kAbsent) pr.at[i] = (pr.at[i] + odd_rows) & ~3u;
                if (pc.at[i] != kAbsent) pc.at[i] = (pc.at[i] + (i < 2 ? odd_cols : odd_second)) & ~3u;
            }
        }
        const unsigned odd_ld_rows = ODD ? t.ld_rows & 1 : 0, odd_ld_cols = ODD ? t.ld_cols & 1 : 0;
        const unsigned shift_rows = ((odd_rows / 2 + (s & odd_ld_rows)) & 1u) * 16u;
        const unsigned shift_cols = ((odd_cols / 2 + (s & odd_ld_cols)) & 1u) * 16u;
        const unsigned shift_second = ((odd_second / 2 + (s & odd_ld_cols)) & 1u) * 16u;

        const unsigned lds0 = lds_address(s_tiles) + wave * 1024;
        // The stage that is being loaded: what it is from, where it goes, and its steps.
        struct Source {
            u32x4 rows, cols, second;
            unsigned to;
            int left;
        };
        auto source = [&](int n, int slot) {
            Source from;
            from.rows = operand_words<L>(t.rows + n * t.step_rows, a.rows_end);
            from.cols = operand_words<L>(t.cols + n * t.step_cols, a.cols_end);
            from.second = GATED ? operand_words<L>(t.second + n * t.step_cols, a.cols_end) : from.cols;
            from.to = lds0 + slot * kStage;
            from.left = t.depth - n * kStep + ODD;  // may be below 1
            return from;
        };
        // Load i of a stage, the rows' first, in three steps that products come between.
        auto load_offset = [&](auto i, const Source& from) {
            if constexpr (i.value < kRowLoads) return pr.template offset<i.value>(from.left);
            else return pc.template offset<i.value - kRowLoads>(from.left);
        };
        auto load_to = [&](auto i, const Source& from) {
            constexpr int at = i.value < kRowLoads ? i.value * 4096 : kRowBytes + (i.value - kRowLoads) * 4096;
            lds_dma_raw_to<at>(from.to);
        };
        auto load_from = [&](auto i, const Source& from, unsigned offset) {
            lds_dma_raw_x4(i.value < kRowLoads ? from.rows : i.value < kRowLoads + 2 ? from.cols : from.second,
                           offset);
        };
        Operand<T> fr[2][RF], fc[2][CF];
        WordPiece raw[2][ODD ? RF + CF : 1];  // Odd: what the operands are shifted from
        // Sixteen rows from n0 on of an operand in `slot`.
        auto read = [&](auto m, int slot, int next, int half) {
            constexpr bool COLS = m.value >= RF;
            using Op = std::conditional_t<COLS, Cols, Rows>;
            const int n0 = COLS ? column(m.value - RF) : (wr * RF + m.value) * 16;
            const char* at = s_tiles + slot * kStage + (COLS ? kRowBytes : 0);
            if constexpr (!ODD) {
                const Operand<T> x = Op::read(reinterpret_cast<const T*>(at), n0, half);
                if constexpr (COLS) fc[half][m.value - RF] = x;
                else fr[half][m.value] = x;
            } else {
                const int c = 4 * half + q, row = (n0 + s) * kStep * 2;
                const char* behind = c == 7 ? s_tiles + next * kStage + (COLS ? kRowBytes : 0) : at;
                raw[half][m.value].words = *reinterpret_cast<const uint4*>(at + row + (c ^ (s & 7)) * 16);
                raw[half][m.value].next =
                    *reinterpret_cast<const unsigned*>(behind + row + (((c + 1) & 7) ^ (s & 7)) * 16);
            }
        };
        // Read m of a half: the rows' operands, then the columns'.
        auto read_one = [&](auto m, int slot, int next, int half) {
            if constexpr (m.value < RF + CF) read(m, slot, next, half);
        };
        // Odd: operand m from its words.
        auto shift_one = [&](auto m, int half) {
            constexpr bool COLS = m.value >= RF;
            const unsigned shift = !COLS ? shift_rows
                                   : GATED && m.value - RF >= CF / 2 ? shift_second : shift_cols;
            Operand<T> x = __builtin_bit_cast(Operand<T>, piece_of(raw[half][m.value], shift / 8));
            asm volatile("" : "+v"(x));
            if constexpr (COLS) fc[half][m.value - RF] = x;
            else fr[half][m.value] = x;
        };
        // The stage whose rows end inside a piece, -1 for none, and what cuts them there: a
        // thread a row.  Odd: a row that begins between two words goes one element further,
        // for which the last stage may have one behind it.
        const int last = t.depth - (stages - 1) * kStep;
        const int partial = L == Lie::Pieces || (GRAD && L == Lie::Words) ? -1
                            : ODD && last == kStep ? stages
                            : ODD || last % 8 != 0 ? stages - 1 : -1;
        auto cut = [&](int slot) {
            const int left = partial == stages ? 0 : last, n = threadIdx.x & 127;
            const bool of_cols = threadIdx.x >= 128;
            if (of_cols ? !COLS_MAJOR : n < BR) {
                char* row = s_tiles + slot * kStage + (of_cols ? kRowBytes : 0) + n * kStep * 2;
                // values, not places: a choice between members would put t into memory
                const int row_further = (odd_rows / 2 + (n & odd_ld_rows)) & 1;
                const int col_further = ((GATED && n >= 64 ? odd_second : odd_cols) / 2 + (n & odd_ld_cols)) & 1;
                const int further = of_cols ? col_further : row_further;
                uint4* piece = reinterpret_cast<uint4*>(row + ((left / 8) ^ (n & 7)) * 16);
                *piece = first_of(*piece, left % 8 + further);
            }
            __syncthreads();
        };
        // A half's products; behind product m, f(m).
        constexpr int kProducts = CF * RF;
        auto multiply = [&](int half, auto f) {
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (ODD) {
                unrolled(std::make_integer_sequence<int, RF + 1>{}, [&](auto m) { shift_one(m, half); });
                // what the vector unit wrote can be read two cycles later, which the compiler
                // would see to for its own products
                asm volatile("s_nop 3");
            }
            unrolled(std::make_integer_sequence<int, kProducts>{}, [&](auto m) {
                mfma_in_place(acc[m.value / RF][m.value % RF], fc[half][m.value / RF], fr[half][m.value % RF]);
                f(m);
                if constexpr (ODD && m.value % RF == 0 && m.value / RF + 1 < CF) {
                    shift_one(std::integral_constant<int, RF + m.value / RF + 1>{}, half);
                    if constexpr (RF < 4) asm volatile("s_nop 1");
                }
                __builtin_amdgcn_sched_barrier(0);
            });
        };
#pragma unroll
        for (int n = 0; n < S; ++n) {
            const Source from = source(n, n);
            unrolled(std::make_integer_sequence<int, kLoads>{}, [&](auto i) {
                load_to(i, from);
                asm volatile("s_nop 0");
                load_from(i, from, load_offset(i, from));
            });
        }
        wait_vmcnt<kLoads * (S - kAhead + 1)>();
        lds_barrier();
        int slot = 0, next = 1;
        // stages 0 (Odd: and 1) are there
        if (L != Lie::Pieces && partial >= 0 && partial <= kAhead - 2) cut(partial);
        unrolled(std::make_integer_sequence<int, RF + CF>{}, [&](auto m) { read_one(m, 0, 1, 0); });
        for (int n = 0; n < stages; ++n) {
            const int after = next + 1 < S ? next + 1 : 0;
            multiply(0, [&](auto m) { read_one(m, slot, next, 1); });
            wait_vmcnt<kLoads * (S - kAhead)>();
            lds_barrier();
            if (L != Lie::Pieces && partial == n + kAhead - 1) cut(ODD ? after : next);
            const Source from = source(n + S, slot);
            unsigned offset[2];
            multiply(1, [&](auto m) {
                // past the last stage there are zeros to read
                read_one(m, next, after, 0);
                constexpr int kEach = kProducts / kLoads;  // products a load: 2, or 1 and all steps at once
                if constexpr (kEach >= 2) {
                    if constexpr (m.value % 2 == 0) {
                        offset[0] = load_offset(std::integral_constant<int, m.value / 2>{}, from);
                        load_to(std::integral_constant<int, m.value / 2>{}, from);
                    } else {
                        load_from(std::integral_constant<int, m.value / 2>{}, from, offset[0]);
                    }
                } else if constexpr (m.value < kLoads) {
                    load_to(m, from);
                    offset[1] = load_offset(m, from);
                    asm volatile("s_nop 0");
                    load_from(m, from, offset[1]);
                }
            });
            slot = next;
            next = after;
        }
        settle_sums(acc);
        wait_vmcnt<0>();
        lds_barrier();  // the ring is free
    }
    static_assert(4 * kLeaveFloats<T, CF, E, RF> * sizeof(float) <= kRingLds, "LDS of the ends");
    leave<T, RF, CF, E, RF>(a, t, r0, c0, acc, s_tiles, wave);
}

// Sums of a wave's share of the contraction for CF x 16 columns (rows of `cols`,
// `width` of them from its first) and RF x 16 rows (of `rows`, `rows_here`), all
// with `depth` contiguous elements: wave w of WAVES takes every WAVES-th 64 steps.
// Operands come straight from memory, as the words around each piece; 64 steps' loads
// are under way (with 128, fewer workgroups a CU: 50 rows x 8000 x 1002 15 us, 10 so).
template <typename T, int RF, int CF, int WAVES, int PARTS = 1>
__device__ __forceinline__ void wave_share(const T* rows, int rows_here, const T* cols, int width,
                                           int depth, Sums<T> (&acc)[CF][RF],
                                           const T* second = nullptr) {
    constexpr int kHere = CF / PARTS;  // 16s of columns of a part
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int s = lane & 15, q = lane >> 4;
    const unsigned odd_r = static_cast<unsigned>(reinterpret_cast<uintptr_t>(rows)) & 2u;
    const unsigned odd_c = static_cast<unsigned>(reinterpret_cast<uintptr_t>(cols)) & 2u;
    const __amdgpu_buffer_rsrc_t br = words_buffer(rows, static_cast<long long>(rows_here) * depth);
    const long long words = static_cast<long long>(min(width, kHere * 16)) * depth;
    const __amdgpu_buffer_rsrc_t bc = words_buffer(cols, words);
    const unsigned odd_s = PARTS == 2 ? static_cast<unsigned>(reinterpret_cast<uintptr_t>(second)) & 2u : 0u;
    const __amdgpu_buffer_rsrc_t bs = PARTS == 2 ? words_buffer(second, words) : bc;
    unsigned ar[RF], ac[CF];  // byte offsets of the first piece; rows past the end are zeros
#pragma unroll
    for (int i = 0; i < RF; ++i) {
        const int r = i * 16 + s;
        ar[i] = r < rows_here ? static_cast<unsigned>(r * depth + 8 * q) * 2u + odd_r : kAbsent;
    }
#pragma unroll
    for (int j = 0; j < CF; ++j) {
        const int c = j % kHere * 16 + s;
        ac[j] = c < width ? static_cast<unsigned>(c * depth + 8 * q) * 2u + (j < kHere ? odd_c : odd_s)
                          : kAbsent;
    }
    auto run = [&](auto odd) {
        for (int k = wave * 64; k < depth; k += WAVES * 64) {
            WordPiece vr[2][RF], vc[2][CF];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int at = k + 32 * half;
                const bool in = at + 8 * q < depth;
#pragma unroll
                for (int j = 0; j < CF; ++j) {
                    vc[half][j] = load_words<odd.value>(j < kHere ? bc : bs, in ? ac[j] + 2u * at : kAbsent);
                }
#pragma unroll
                for (int i = 0; i < RF; ++i) {
                    vr[half][i] = load_words<odd.value>(br, in ? ar[i] + 2u * at : kAbsent);
                }
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int left = depth - k - 32 * half;
                auto operand = [&](const WordPiece& v, unsigned byte) {
                    uint4 x = odd.value ? piece_of(v, byte) : v.words;
                    if (left < 32) x = first_of(x, left - 8 * q);
                    return __builtin_bit_cast(Operand<T>, x);
                };
                Operand<T> fr[RF];
#pragma unroll
                for (int i = 0; i < RF; ++i) fr[i] = operand(vr[half][i], ar[i]);
#pragma unroll
                for (int j = 0; j < CF; ++j) {
                    const Operand<T> fc = operand(vc[half][j], ac[j]);
#pragma unroll
                    for (int i = 0; i < RF; ++i) acc[j][i] = mfma(fc, fr[i], acc[j][i]);
                }
            }
        }
    };
    // rows that begin between two words, or not
    if (((odd_r | odd_c | odd_s) & 2u) != 0 || (depth & 1) != 0) run(std::true_type{});
    else run(std::false_type{});
}

// wave_share for operands whose rows are whole 16-byte pieces (the same sums in the
// same order): a wave's pieces go through a ring of D stages of LDS of its own (no
// barriers).  A load then brings eight rows' whole cache lines; operands read
// straight from memory are 64 bytes of sixteen rows, which the cache serves more
// slowly (8 groups of 4000 columns, 32 rows: 4096 steps 42 us, 4098 47).
//   ring: WAVES x D x (RF + CF) x 2 KB.
template <typename T, int RF, int CF, int WAVES, int D, int PARTS = 1>
__device__ __forceinline__ void ring_share(char* ring, const T* rows, int rows_here, const T* cols,
                                           int width, int depth, Sums<T> (&acc)[CF][RF],
                                           const T* second = nullptr) {
    constexpr int kHere = 2 * CF / PARTS;  // loads of a part
    constexpr int kLoads = 2 * (RF + CF), kStage = kLoads * 1024;
    static_assert(kLoads * (D - 1) < 64, "vmcnt is 6 bits");
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int s = lane & 15, q = lane >> 4;
    // load i brings rows 8 i .. 8 i + 7; piece p of a row is at place p ^ (row & 7)
    const int piece = (lane & 7) ^ (lane >> 3);
    unsigned at_col[2 * CF], at_row[2 * RF];
#pragma unroll
    for (int i = 0; i < 2 * CF; ++i) {
        const int n = 8 * (i % kHere) + (lane >> 3);
        at_col[i] = n < width ? static_cast<unsigned>(n * depth + piece * 8) * 2u : kAbsent;
    }
#pragma unroll
    for (int i = 0; i < 2 * RF; ++i) {
        const int n = 8 * i + (lane >> 3);
        at_row[i] = n < rows_here ? static_cast<unsigned>(n * depth + piece * 8) * 2u : kAbsent;
    }
    const unsigned lds0 = lds_address(ring) + wave * D * kStage;
    const char* own = ring + wave * D * kStage;
    const int stages = ((depth + 63) / 64 - wave + WAVES - 1) / WAVES;  // may be 0
    auto load = [&](int n, int slot) {
        const int k = (n * WAVES + wave) * 64;
        const bool in = piece * 8 < depth - k;  // past the end: zeros
        const u32x4 bc = buffer_words(cols + k, 0, 0x7fffffff);
        const u32x4 bs = PARTS == 2 ? buffer_words(second + k, 0, 0x7fffffff) : bc;
        const u32x4 br = buffer_words(rows + k, 0, 0x7fffffff);
        unrolled(std::make_integer_sequence<int, 2 * CF>{}, [&](auto i) {
            lds_dma_raw_to<i.value * 1024>(lds0 + slot * kStage);
            asm volatile("s_nop 0");
            lds_dma_raw_x4(i.value < kHere ? bc : bs, in ? at_col[i.value] : kAbsent);
        });
        unrolled(std::make_integer_sequence<int, 2 * RF>{}, [&](auto i) {
            lds_dma_raw_to<(2 * CF + i.value) * 1024>(lds0 + slot * kStage);
            asm volatile("s_nop 0");
            lds_dma_raw_x4(br, in ? at_row[i.value] : kAbsent);
        });
    };
#pragma unroll
    for (int n = 0; n < D - 1; ++n) load(n, n);
    int slot = 0, to = D - 1;
    for (int n = 0; n < stages; ++n) {
        load(n + D - 1, to);
        wait_vmcnt<kLoads * (D - 1)>();
        asm volatile("" ::: "memory");  // reads below, not before
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            Operand<T> fr[RF], fc[CF];
            auto read = [&](int tile) {
                return *reinterpret_cast<const Operand<T>*>(
                    own + slot * kStage + tile * 2048 + s * 128 + ((4 * half + q) ^ (s & 7)) * 16);
            };
#pragma unroll
            for (int j = 0; j < CF; ++j) fc[j] = read(j);
#pragma unroll
            for (int i = 0; i < RF; ++i) fr[i] = read(CF + i);
#pragma unroll
            for (int j = 0; j < CF; ++j)
#pragma unroll
                for (int i = 0; i < RF; ++i) acc[j][i] = mfma(fc[j], fr[i], acc[j][i]);
        }
        // the slot's reads are done before the next load may overwrite it
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        slot = slot + 1 < D ? slot + 1 : 0;
        to   = to + 1 < D ? to + 1 : 0;
    }
    wait_vmcnt<0>();
}

// Adds the waves' shares up in LDS in a fixed order: afterwards total(c, r) is the
// sum for column c and row r of the workgroup's tile.
template <int RF, int CF, int WAVES, typename V = f32x4>
struct Shares {
    static constexpr int kBytes = WAVES * CF * RF * 1024;
    using Sum = std::conditional_t<std::is_same_v<V, i32x4>, int, float>;
    Sum (*parts)[CF][RF][64][4];
    __device__ __forceinline__ explicit Shares(char* lds)
        : parts(reinterpret_cast<Sum (*)[CF][RF][64][4]>(lds)) {}
    __device__ __forceinline__ void put(const V (&acc)[CF][RF]) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
        for (int j = 0; j < CF; ++j)
#pragma unroll
            for (int i = 0; i < RF; ++i) *reinterpret_cast<V*>(parts[wave][j][i][lane]) = acc[j][i];
    }
    __device__ __forceinline__ Sum total(int c, int r) const {
        Sum sum = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            sum += parts[w][c / 16][r / 16][(c % 16) / 4 * 16 + r % 16][c % 4];
        }
        return sum;
    }
};

// The ends of few_rows_product: a thread takes a column's sums of some rows.
template <typename T, Ends E, int CF, int WAVES, typename S>
__device__ __forceinline__ void add_few(const TileArgs& a, const RowTile& t, int c0, const S& shares) {
    const int rows_here = t.end - t.first;
    T* out = static_cast<T*>(a.out) + static_cast<long long>(t.first) * a.width;
    const int c = threadIdx.x % (CF * 16);
    if (c0 + c >= a.width) return;
    for (int s = threadIdx.x / (CF * 16); s < rows_here; s += WAVES * 4 / CF) {
        float sum = static_cast<float>(shares.total(c, s));
        if constexpr (E == Ends::Adapters) {
            const int id = a.ids[t.first + s];
            if (static_cast<unsigned>(id) < static_cast<unsigned>(a.adapters)) {
                const float* h = a.h + static_cast<long long>(t.first + s) * a.rank16;
                const T* b = static_cast<const T*>(a.b) +
                             (static_cast<long long>(id) * a.width + c0 + c) * a.rank;
                float part = 0.0f;
                for (int k = 0; k < a.rank; k += 8) {
                    const int n = min(8, a.rank - k);
                    float x[8], y[8];
                    __builtin_memcpy(x, h + k, 32);
                    piece_to_float<T>(n == 8 ? load_piece(b + k) : load_part(b + k, n), y);
#pragma unroll
                    for (int i = 0; i < 8; ++i) part = fmaf(x[i], y[i], part);
                }
                sum += part;
            }
        }
        out[static_cast<long long>(s) * a.width + c0 + c] = static_cast<T>(sum);
    }
}
template <typename T, bool GATED, int OUT, int WAVES, typename S>
__device__ __forceinline__ void finish_few(const TileArgs& a, const RowTile& t, bool grouped, int c0,
                                           const S& shares) {
    constexpr int  PARTS = GATED ? 2 : 1;
    constexpr bool kScaled = std::is_same_v<T, Int8Pair>;
    const int c = threadIdx.x % OUT, rows_here = t.end - t.first;
    if (c0 + c >= a.width) return;
    float scale[PARTS] = {};
    if (kScaled && grouped) {
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            scale[part] = a.col_scales[(static_cast<long long>(t.group) * PARTS + part) * a.width + c0 + c];
        }
    }
    for (int s = threadIdx.x / OUT; s < rows_here; s += WAVES * 64 / OUT) {
        const long long row = static_cast<long long>(t.first) + s;
        float f[PARTS];
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            f[part] = static_cast<float>(shares.total(part * OUT + c, s));
            if (kScaled && grouped) f[part] = f[part] * scale[part] * a.row_scales[row];
            if constexpr (GATED && !kScaled) {
                if (a.kept != nullptr) {
                    static_cast<T*>(a.kept)[(2 * row + part) * a.width + c0 + c] = static_cast<T>(f[part]);
                }
            }
        }
        float h = f[0];
        if constexpr (GATED) h = gate_value(a.act, f[0]) * f[PARTS - 1];
        if constexpr (kScaled) store_as(a.out, a.out_type, row * a.width + c0 + c, h);
        else static_cast<T*>(a.out)[row * a.width + c0 + c] = static_cast<T>(h);
    }
}

// Products of few rows, bound by reading the weights (W [c][k]) once: a workgroup
// takes CF x 16 columns and up to RF x 16 rows of a group, its waves share the
// contraction, so that a projection of a few thousand columns still has a workgroup
// a CU.  D: as for adapter_shrink.  64 groups of 2048 x 4096, 256 rows: 168 us, 6.4 TB/s,
// what reads alone reach; 48 rows x 4096 x 4096 with adapters 10.5 us.
//   Gated: half of the columns are the gates, half what they multiply.
template <typename T, int RF, int CF, int WAVES, int D, bool GATED, bool ADAPT>
__global__ __launch_bounds__(WAVES * 64) void few_rows_product(TileArgs a) {
    extern __shared__ __attribute__((aligned(16))) char s_ring[];  // and then the shares
    constexpr Ends E = GATED ? Ends::Gated : ADAPT ? Ends::Adapters : Ends::Plain;
    constexpr int PARTS = GATED ? 2 : 1, OUT = CF * 16 / PARTS;
    const int col_tiles = (a.width + OUT - 1) / OUT;
    const RowTile t = find_tile<RF * 16>(a, blockIdx.x / col_tiles);
    if (t.group < 0) return;
    const int c0 = blockIdx.x % col_tiles * OUT;
    const int rows_here = t.end - t.first;
    const bool grouped = t.group < a.groups;  // rows in no group: zeros
    Sums<T> acc[CF][RF];
#pragma unroll
    for (int j = 0; j < CF; ++j)
#pragma unroll
        for (int i = 0; i < RF; ++i) acc[j][i] = Sums<T>(0);
    if (grouped) {
        const T* x = static_cast<const T*>(a.rows) + static_cast<long long>(t.first) * a.depth;
        const T* w = static_cast<const T*>(a.cols) +
                     (static_cast<long long>(t.group) * PARTS * a.width + c0) * a.depth;
        const T* w2 = GATED ? w + static_cast<long long>(a.width) * a.depth : nullptr;
        if constexpr (D > 0) {
            ring_share<T, RF, CF, WAVES, D, PARTS>(s_ring, x, rows_here, w, a.width - c0, a.depth, acc, w2);
            __syncthreads();
        } else {
            wave_share<T, RF, CF, WAVES, PARTS>(x, rows_here, w, a.width - c0, a.depth, acc, w2);
        }
    }
    Shares<RF, CF, WAVES, Sums<T>> shares(s_ring);
    shares.put(acc);
    __syncthreads();
    if constexpr (!kPlainEnds<T, E>) {
        finish_few<T, GATED, OUT, WAVES>(a, t, grouped, c0, shares);
    } else {
        add_few<T, E, CF, WAVES>(a, t, c0, shares);
    }
}

// The largest extent that 32-bit element offsets inside a tile reach.
constexpr long long kMostElements = 1LL << 30;

Error check_product(int total, int groups, int width, int depth, const char* name) {
    if (total < 0 || groups < 1 || width < 1 || depth < 1) {
        return Error{kInvalid, std::string(name) + ": sizes must be positive"};
    }
    if (256LL * std::max(width, depth) > kMostElements) {
        return Error{kUnsupported, std::string(name) + ": rows over 2^22 elements"};
    }
    // a tile past the last row has to stay an int
    if (total > 0x7fff0000) {
        return Error{kUnsupported, std::string(name) + ": over 2^31 - 2^16 rows"};
    }
    return Error{};
}

template <typename F>
Error with_half(ElementType type, const char* name, F f) {
    if (type == ElementType::F16) return f(_Float16{});
    if (type == ElementType::BF16) return f(__bf16{});
    return Error{kUnsupported, std::string(name) + ": fp16 or bf16 operands (matrix cores)"};
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Refuses a launch that HIP would drop.
Error check_threads(long long blocks, int threads, const char* name) {
    if (blocks * threads <= kLaunchThreads) return Error{};
    return Error{kUnsupported, std::string(name) + ": the launch would need 2^32 threads or more"};
}

constexpr int kWideLds   = 10 * 128 * kStep * 2;      // ten slots
constexpr int kSharedLds = 4 * 2 * 128 * kStep * 2;  // four groups' two buffers

// Launches kernel with `lds` bytes of dynamic LDS, asked for once a GPU.
template <auto kernel, typename... Args>
Error launch_with_lds(dim3 grid, int threads, int lds, hipStream_t stream, const char* name,
                      Args... args) {
    static OncePerDevice grown;
    const auto ask = [&] {
        return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                   hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    };
    SPMM_TRY_HIP(grown(ask), name);
    kernel<<<grid, threads, lds, stream>>>(args...);
    SPMM_TRY_HIP(hipGetLastError(), name);
    return Error{};
}

// Stages of a ring of `waves` waves with a stage of `tiles` x 2 KB within `room`
// bytes; the waves' shares fit in it too.
constexpr int ring_depth(int waves, int tiles, int room) {
    return std::min(8, room / (waves * tiles * 2048));
}

template <typename T, int RF, int CF, int WAVES, int ROOM, Ends E>
Error launch_few_rows_of(const TileArgs& a, bool pieces, hipStream_t stream, const char* name) {
    constexpr bool gated = E == Ends::Gated, adapt = E == Ends::Adapters;
    constexpr int OUT = gated ? CF * 8 : CF * 16;
    const long long row_tiles = a.offsets == nullptr
        ? (a.total + RF * 16 - 1) / (RF * 16)
        : a.total / (RF * 16) + std::min<long long>(a.groups + 2LL, a.total);
    const long long blocks = row_tiles * ((a.width + OUT - 1) / OUT);
    SPMM_TRY(check_threads(blocks, WAVES * 64, name));
    const dim3 grid(static_cast<unsigned>(blocks));
    constexpr int shares = Shares<RF, CF, WAVES>::kBytes;
    if constexpr (CF == (gated ? 2 : 1) && !std::is_same_v<T, Int8Pair>) {
        if (!pieces) {
            return launch_with_lds<few_rows_product<T, RF, CF, WAVES, 0, gated, adapt>>(
                grid, WAVES * 64, shares, stream, name, a);
        }
    }
    constexpr int depth = ring_depth(WAVES, RF + CF, ROOM);
    constexpr int lds = std::max(shares, WAVES * depth * (RF + CF) * 2048);
    return launch_with_lds<few_rows_product<T, RF, CF, WAVES, depth, gated, adapt>>(
        grid, WAVES * 64, lds, stream, name, a);
}
// Rows of a group that few_rows_product is launched for: all of one group's, and twice the
// mean of more, so that few of them need a second tile that reads W again.
long long few_rows(const TileArgs& a) {
    const long long groups = a.offsets == nullptr ? 1 : std::min(a.groups, a.total);
    return groups == 1 ? a.total : 2LL * a.total / groups;
}
// How few_rows_product is launched for gated products and for those in 8-bit integers: four
// waves and two workgroups a CU with sixteen columns of either projection, or 32 (rows of
// integers are half as long, and the rows' own reading counts twice as much: 64 groups of
// 2048 x 4096, 256 rows 93 us, 107 with sixteen columns; a single group has the workgroups to
// hide that: 8192 x 8192, 16 rows 15.4, 19.9 with 32).  All of the LDS where there is one
// workgroup a CU and its rows leave no stages else (gated, 2 x 1024 x 4096, 64 rows: 15 us, 20).
template <typename T, Ends E>
Error launch_few_finished(const TileArgs& a, bool pieces, hipStream_t stream, const char* name) {
    constexpr int kTwo = 80 * 1024, kAll = 160 * 1024;
    const long long rows = few_rows(a);
    if constexpr (E == Ends::Gated) {
        const long long row_tiles = a.offsets == nullptr ? (a.total + 63) / 64 : a.groups;
        if (rows <= 16) return launch_few_rows_of<T, 1, 2, 4, kTwo, E>(a, pieces, stream, name);
        if (rows <= 32) return launch_few_rows_of<T, 2, 2, 4, kTwo, E>(a, pieces, stream, name);
        if (pieces && row_tiles * ((a.width + 15) / 16) <= 256) {
            return launch_few_rows_of<T, 4, 2, 4, kAll, E>(a, pieces, stream, name);
        }
        return launch_few_rows_of<T, 4, 2, 4, kTwo, E>(a, pieces, stream, name);
    } else if (a.offsets == nullptr || a.groups == 1) {
        if (rows <= 16) return launch_few_rows_of<T, 1, 1, 4, kTwo, E>(a, pieces, stream, name);
        if (rows <= 32) return launch_few_rows_of<T, 2, 1, 4, kTwo, E>(a, pieces, stream, name);
        return launch_few_rows_of<T, 4, 1, 4, kTwo, E>(a, pieces, stream, name);
    } else {
        if (rows <= 16) return launch_few_rows_of<T, 1, 2, 4, kTwo, E>(a, pieces, stream, name);
        if (rows <= 32) return launch_few_rows_of<T, 2, 2, 4, kTwo, E>(a, pieces, stream, name);
        if (a.groups * static_cast<long long>((a.width + 31) / 32) <= 256) {
            return launch_few_rows_of<T, 4, 2, 4, kAll, E>(a, pieces, stream, name);
        }
        return launch_few_rows_of<T, 4, 2, 4, kTwo, E>(a, pieces, stream, name);
    }
}
// The kernels a product can take: few_rows_product, tile_product through registers
// or with pieces straight into LDS, tile_product_wide, tile_product_shared, tile_product_ring
// of 64 or 128 rows.
enum class Form { FewRows, Any, Pieces, Wide, Shared, Ring64, Ring128 };
constexpr int threads_of(Form form) { return form == Form::Shared ? 1024 : 256; }
constexpr int edge_of(Form form) { return form == Form::Wide ? 256 : form == Form::Shared ? 64 : 128; }
constexpr int rows_of(Form form) { return form == Form::Ring64 ? 64 : edge_of(form); }

// Estimated microseconds of a form for `row_tiles(edge)` x width tiles of `steps`
// steps, from measured rates: 64 steps of a 128 x 128 tile take 0.62 us where a CU has
// one and 0.95 us where it has two (through registers 1 and 1.5 us), of a 256 x 256 tile
// 1.55 us, one a CU, and 256 steps of a 64 x 64 tile 1.1 us, one a CU; of the ring's tiles,
// one a CU, 64 steps of 64 x 128 take 0.48 us and of 128 x 128 0.62; `weights` microseconds is
// what reading the weights takes.
template <typename F>
double tile_time(Form form, F row_tiles, int width, double steps, double weights) {
    const int edge = edge_of(form);
    const double tiles = row_tiles(edge) * std::ceil(static_cast<double>(width) / edge);
    if (tiles * threads_of(form) > kLaunchThreads) return HUGE_VAL;
    const double rounds = std::ceil(steps / kStep);
    if (form == Form::Shared) {
        return std::max(std::ceil(tiles / 256) * (4 + 1.1 * std::ceil(rounds / 4)), weights);
    }
    if (form == Form::Wide) {
        return std::max(std::ceil(tiles / 256) * (6 + 1.55 * rounds), weights);
    }
    if (form == Form::Ring128) {
        return std::max(std::ceil(tiles / 256) * (3 + 0.62 * rounds), weights);
    }
    if (form == Form::Ring64) {  // row_tiles counts its rows
        const double low = row_tiles(64) * std::ceil(width / 128.0);
        return std::max(std::ceil(low / 256) * (3 + 0.48 * rounds), weights);
    }
    const double two = form == Form::Any ? 1.5 : 0.95, one = form == Form::Any ? 1 : 0.62;
    const double whole = std::floor(tiles / 512), rest = tiles - 512 * whole;
    const double time = whole * (3 + two * rounds) +
                        (rest == 0 ? 0 : 3 + (rest <= 256 ? one : two) * rounds);
    return std::max(time, weights);
}
// How a product's operands lie (x and w: all rows of both).
inline Lie lie_of(const TileArgs& a, long long ld_rows, long long ld_cols) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.rows) | reinterpret_cast<uintptr_t>(a.cols);
    const long long ld = ld_rows | ld_cols;
    return ld % 8 == 0 && at % 16 == 0 ? Lie::Pieces : ld % 2 == 0 && at % 4 == 0 ? Lie::Words : Lie::Odd;
}

// Microseconds of `tiles` tiles of 256 x 256 with `rounds` x 64 steps that end gated or scaled.
inline double finished_wide(double tiles, double rounds) {
    return 4 + std::ceil(tiles / 256) * (11 + 1.45 * rounds);
}
// The form of a gated product or one in 8-bit integers (whose depth is in pairs), by its
// estimated time, from measured rates; width: rows of a group's weights, of both projections
// of a gated one; gated: 16 columns of either a workgroup of few_rows_product.
//   few_rows_product: weights at 6.3 TB/s, more slowly as the rows' own reading counts and
//     where a second tile of rows reads them again, the rows themselves, which each of its
//     workgroups reads, at 12; 512 workgroups at a time, which take 3 us
//     and for 1000 steps 1.4 us with 16 rows, 2.6 with 64, 5.5 where those leave no stages
//     ahead (2 x 8192 x 4096: 16 rows 27 us, 64 36, 128 59; 2 x 1024 x 2048: 16 rows 5.0, 256
//     8.6; 8 groups of 2 x 7552 x 304 in integers, 21 rows: 24, 16 in tile_product).  1.1 times
//     as long for rows that are no whole pieces, twice where they begin between two words.
//   tile_product_ring: 64 steps of a 64 x 128 tile take 0.42 us, of 128 x 128 0.57, more where
//     rows are cut or shifted, one tile a CU; weights at 3.5 TB/s (2 x 8192 x 4096: 128 rows
//     39 and 49 us, 256 68 and 49; tile_product 62, 68).
//   tile_product: 0.85 us with one tile a CU, 1.15 with two, through registers 1.2 and 1.5;
//     tile_product_wide 1.45 and 11 us for a tile's beginning and end (2 x 8192 x 4096: 512
//     rows 79 us in tile_product, 88 in the ring, 1024 rows 113 wide, 154 and 167; 24771 rows x
//     2 x 2430 x 160: 97 in tile_product, 125 wide).
inline Form choose_finished(const TileArgs& a, int width, bool gated, Lie lie, bool packs, double* time) {
    const double groups = a.offsets == nullptr ? 1 : std::min(a.groups, a.total);
    const double mean = a.total / groups, weights = 2.0 * groups * width * a.depth;
    // groups of all lengths end, on average, in the middle of a tile
    auto row_tiles = [&](int edge) {
        return groups == 1 ? std::ceil(mean / edge) : groups * std::max(1.0, mean / edge + 0.5);
    };
    const int l = static_cast<int>(lie);
    const double rounds = std::ceil(static_cast<double>(a.depth) / kStep);
    auto ring = [&](Form f, double begin, double stage) {
        const double high = row_tiles(rows_of(f));
        // a few tiles more than groups have on average may be another round
        const double more = groups == 1 ? 0 : std::min(0.1, 0.3 * groups / high);
        const double tiles = high * std::ceil(width / 128.0) * (1 + more);
        if (tiles * 256 > kLaunchThreads) return HUGE_VAL;
        return std::max(2 + std::ceil(tiles / 256) * (begin + stage * rounds), weights / 3.5e6);
    };
    constexpr double stage64[] = {0.42, 0.48, 0.75}, stage128[] = {0.57, 0.62, 0.9};
    double best = ring(Form::Ring64, 3, stage64[l]);
    Form form = Form::Ring64;
    auto take = [&](Form f, double time) {
        if (time < best) {
            best = time;
            form = f;
        }
    };
    take(Form::Ring128, ring(Form::Ring128, 4.5, stage128[l]));
    const double tiles = row_tiles(128) * std::ceil(width / 128.0);
    if (tiles * 256 <= kLaunchThreads) {
        const double one = lie != Lie::Odd ? 0.85 : 1.2, two = lie != Lie::Odd ? 1.15 : 1.5;
        const double whole = std::floor(tiles / 512), rest = tiles - 512 * whole;
        take(lie != Lie::Odd ? Form::Pieces : Form::Any,
             std::max(2 + whole * (4 + two * rounds) +
                          (rest == 0 ? 0 : 3.5 + (rest <= 256 ? one : two) * rounds),
                      weights / 3.5e6));
    }
    if (lie != Lie::Odd) {
        const double wide = row_tiles(256) * std::ceil(width / 256.0);
        if (wide * 256 <= kLaunchThreads) {
            take(Form::Wide, std::max(finished_wide(wide, rounds), weights / 3.5e6));
        }
    }
    if (!packs) {
        const double again = row_tiles(64) / groups, rows = std::min<double>(few_rows(a), 64.0);
        const double slower = std::max(1 + mean / 160, again > 1 ? 1.15 * again : 0.0);
        const double reading = std::max(weights / 6.3e6 * slower, a.total / 6e6 * a.depth * (width / 32.0));
        const double workgroups = row_tiles(64) * std::ceil(width / (gated || groups > 1 ? 32.0 : 16.0));
        const double ahead = rows <= 32 || workgroups <= 256 ? 1 + rows / 40 : 5.5;
        take(Form::FewRows,
             (1.3 + std::max(2 + reading, std::ceil(workgroups / 512) * (3 + a.depth / 1000.0 * ahead))) *
                 (lie == Lie::Pieces ? 1 : lie == Lie::Words ? 1.1 : 2));
    }
    *time = best;
    return form;
}

// How many of `rows` output rows (a group's, of `groups` as high as each other) go to 256 x
// 256 tiles in whole rounds of a tile a CU, the rest to what is fastest for it: 0 for none, or
// where one launch takes no longer.  time(rows, form): the best form's estimate, or with a
// form that one's (8192 rows for 11264 x 2048, 352 tiles: 256 and 384 of 128 x 128 346 us,
// 356 in one launch; 9000 for 2 x 1024 x 4096, gated: 139 us, 180).
template <typename F>
int whole_rounds(int rows, int groups, int width, F time) {
    const long long col_tiles = (width + 255) / 256, tiles = groups * ((rows + 255) / 256) * col_tiles;
    const long long high = tiles / 256 * 256 / (groups * col_tiles);  // row tiles a group
    const int head = static_cast<int>(high * 256);
    if (high < 1 || head >= rows) return 0;
    return time(head, true) + time(rows - head, false) + 2 < 0.93 * time(rows, false) ? head : 0;
}

// A product's rows [first, first + rows) by themselves, of one group that has all.
inline TileArgs rows_alone(const TileArgs& all, int first, int rows, int out_bytes) {
    TileArgs a = all;
    auto later = [&](const void* p, long long bytes) { return static_cast<const char*>(p) + first * bytes; };
    a.total = rows;
    a.rows = later(all.rows, 2LL * all.depth);
    a.out = const_cast<char*>(later(all.out, static_cast<long long>(all.width) * out_bytes));
    if (all.row_scales != nullptr) a.row_scales = all.row_scales + first;
    if (all.kept != nullptr) {
        const bool packed = all.kept_scales != nullptr;
        a.kept = const_cast<char*>(later(all.kept, 2LL * all.width * (packed ? 1 : 2)));
        const long long line = 2LL * ((all.width + kPackBlock - 1) / kPackBlock);
        if (packed) a.kept_scales = all.kept_scales + first * line;
    }
    return a;
}

template <typename T, bool GRAD, bool COLS_MAJOR, Ends E, Lie L, int RF>
Error launch_ring(const TileArgs& a, long long blocks, hipStream_t stream, const char* name) {
    return launch_with_lds<tile_product_ring<T, GRAD, COLS_MAJOR, E, L, RF>>(
        dim3(static_cast<unsigned>(blocks)), 256, kRingLds, stream, name, a);
}

// Launches the tile kernel of a form.
template <typename T, bool GRAD, bool COLS_MAJOR, Ends E>
Error launch_tiles(const TileArgs& a, Form form, Lie lie, hipStream_t stream, const char* name) {
    const int edge = edge_of(form), out = E == Ends::Gated ? edge / 2 : edge, rows = rows_of(form);
    // every group may end in a part-filled tile, and so may the rows before and behind them
    const long long row_tiles =
        GRAD ? static_cast<long long>(a.groups) * ((a.upto - a.from + rows - 1) / rows)
        : a.offsets == nullptr ? (a.total + rows - 1) / rows
                               : a.total / rows + std::min<long long>(a.groups + 2LL, a.total);
    // a whole number of workgroups for each XCD
    const long long blocks = (row_tiles * ((a.width + out - 1) / out) + 7) / 8 * 8;
    SPMM_TRY(check_threads(blocks, threads_of(form), name));
    const dim3 grid(static_cast<unsigned>(blocks));
    constexpr bool kNew = !kPlainEnds<T, E>, kInt = std::is_same_v<T, Int8Pair>;
    if (form == Form::Wide) {
        if constexpr (!kInt && E != Ends::Adapters) {
            if (lie == Lie::Words) {
                return launch_with_lds<tile_product_wide<T, GRAD, COLS_MAJOR, E, Lie::Words>>(
                    grid, threads_of(Form::Wide), kWideLds, stream, name, a);
            }
        }
        return launch_with_lds<tile_product_wide<T, GRAD, COLS_MAJOR, E>>(
            grid, threads_of(Form::Wide), kWideLds, stream, name, a);
    }
    if constexpr (kNew) {
        const bool low = form == Form::Ring64;
        if (low || form == Form::Ring128) {
            if constexpr (!kInt) {
                if (lie == Lie::Words) {
                    return low ? launch_ring<T, false, false, E, Lie::Words, 2>(a, blocks, stream, name)
                               : launch_ring<T, false, false, E, Lie::Words, 4>(a, blocks, stream, name);
                }
                if (lie == Lie::Odd) {
                    return low ? launch_ring<T, false, false, E, Lie::Odd, 2>(a, blocks, stream, name)
                               : launch_ring<T, false, false, E, Lie::Odd, 4>(a, blocks, stream, name);
                }
            }
            return low ? launch_ring<T, false, false, E, Lie::Pieces, 2>(a, blocks, stream, name)
                       : launch_ring<T, false, false, E, Lie::Pieces, 4>(a, blocks, stream, name);
        }
    } else {
        if constexpr (E != Ends::Adapters) {
            if constexpr (!GRAD && COLS_MAJOR) {
                if (form == Form::Ring64) {
                    return lie == Lie::Words
                        ? launch_ring<T, GRAD, COLS_MAJOR, E, Lie::Words, 2>(a, blocks, stream, name)
                        : launch_ring<T, GRAD, COLS_MAJOR, E, Lie::Pieces, 2>(a, blocks, stream, name);
                }
                if (form == Form::Ring128 && lie == Lie::Pieces) {
                    return launch_ring<T, GRAD, COLS_MAJOR, E, Lie::Pieces, 4>(a, blocks, stream, name);
                }
            }
            if (form == Form::Ring128) {
                return launch_ring<T, GRAD, COLS_MAJOR, E, Lie::Words, 4>(a, blocks, stream, name);
            }
        }
        if (form == Form::Shared) {
            return launch_with_lds<tile_product_shared<T, GRAD, COLS_MAJOR, E>>(
                grid, threads_of(Form::Shared), kSharedLds, stream, name, a);
        }
    }
    if constexpr (kInt) {  // whose rows are whole pieces
        tile_product<T, GRAD, COLS_MAJOR, E, Lie::Pieces><<<grid, 256, 0, stream>>>(a);
    } else if (form == Form::Any) {
        tile_product<T, GRAD, COLS_MAJOR, E, Lie::Odd><<<grid, 256, 0, stream>>>(a);
    } else if (lie == Lie::Pieces) {
        tile_product<T, GRAD, COLS_MAJOR, E, Lie::Pieces><<<grid, 256, 0, stream>>>(a);
    } else if constexpr (E != Ends::Adapters) {
        tile_product<T, GRAD, COLS_MAJOR, E, Lie::Words><<<grid, 256, 0, stream>>>(a);
    }
    SPMM_TRY_HIP(hipGetLastError(), name);
    return Error{};
}

// Launches a gated product or one in 8-bit integers, in one or two parts.
template <typename T, Ends E>
Error launch_finished(const TileArgs& a, Lie lie, hipStream_t stream, const char* name) {
    const int width = E == Ends::Gated ? 2 * a.width : a.width;
    const bool packs = a.kept_scales != nullptr;
    auto launch = [&](const TileArgs& part, Form form) {
        if (form == Form::FewRows) return launch_few_finished<T, E>(part, lie == Lie::Pieces, stream, name);
        return launch_tiles<T, false, false, E>(part, form, lie, stream, name);
    };
    double best;
    constexpr bool gated = E == Ends::Gated;
    const Form form = choose_finished(a, width, gated, lie, packs, &best);
    if (a.offsets == nullptr && lie != Lie::Odd) {
        const int bytes = std::is_same_v<T, Int8Pair> && a.out_type == ElementType::F32 ? 4 : 2;
        const int head = whole_rounds(a.total, 1, width, [&](int rows, bool wide) {
            TileArgs part = a;
            part.total = rows;
            double time;
            choose_finished(part, width, gated, lie, packs, &time);
            return wide ? finished_wide(std::ceil(rows / 256.0) * std::ceil(width / 256.0),
                                        std::ceil(static_cast<double>(a.depth) / kStep)) : time;
        });
        if (head > 0) {
            SPMM_TRY(launch(rows_alone(a, 0, head, bytes), Form::Wide));
            const TileArgs rest = rows_alone(a, head, a.total - head, bytes);
            return launch(rest, choose_finished(rest, width, gated, lie, packs, &best));
        }
    }
    return launch(a, form);
}

// The operands of a product in 8-bit integers, checked: depth bytes a row, in pairs.
inline Error int8_args(const void* x, const float* x_scales, const void* w, const float* w_scales,
                       const int* offsets, int groups, int total, int width, int depth,
                       ElementType out_type, void* out, const char* name, TileArgs& a) {
    if (depth % 16 != 0) {
        return Error{kInvalid, std::string(name) + ": rows of whole 16 values (zeros behind the last)"};
    }
    // 128^2 depth has to stay below 2^31
    if (depth > 131056) return Error{kUnsupported, std::string(name) + ": rows over 131056 values"};
    SPMM_TRY(check_product(total, groups, width, depth / 2, name));
    if (total == 0) return Error{};
    if (x == nullptr || x_scales == nullptr || w == nullptr || w_scales == nullptr ||
        (offsets == nullptr && groups != 1) || out == nullptr) {
        return Error{kInvalid, std::string(name) + ": null pointer"};
    }
    if (!aligned16(x) || !aligned16(w)) {
        return Error{kInvalid, std::string(name) + ": values have to be 16-byte aligned"};
    }
    a.rows = x;
    a.cols = w;
    a.out = out;
    a.offsets = offsets;
    a.groups = groups;
    a.total = total;
    a.width = width;
    a.depth = depth / 2;
    a.row_scales = x_scales;
    a.col_scales = w_scales;
    a.out_type = out_type;
    return Error{};
}

}  // namespace
}  // namespace engine
}  // namespace spmm
