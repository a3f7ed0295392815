// Products of rows in group order with their group's weights, and a shared
// projection with each row's low-rank adapter:
//
//   product    out[s, c] = sum_k X[s, k] W_g[c, k]  (or W_g[k, c]),  s in group g
//   gradient   out_g[r, c] = sum_{s in g} P[s, r] Q[s, c]            of the weights
//   adapters   out[s, c] = sum_k X[s, k] W[c, k] + sum_r h[s, r] B_a[c, r],
//              h[s, r] = scale_a sum_k X[s, k] A_a[r, k],  a = ids[s]
//
// The first is the product of a block-diagonal matrix (each group's rows a block)
// with dense weights, and the adapters extend the contraction by a block-sparse
// operand: one block of h a row against the stacked B.  Tile kernels (256 x 256, 128 x
// 128, and 64 x 64 for few tiles with a long contraction) and a kernel for few rows do all
// three on matrix cores (v_mfma_f32_16x16x32, fp32 sums), 64 steps of the contraction at a
// time through LDS.  Many rows are bound by how well the matrix cores are fed and by the
// clock that they leave, few by reading W.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>
#include <utility>

#include "amdgcn.h"
#include "elements.h"
#include "engine.h"
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

// A byte offset past every buffer's 2^31 - 1 bytes, with room for the 16 that a
// load adds: it reads zeros.
constexpr unsigned kAbsent = 0x80000000u;

// A 16-bit element type's operand of one 16x16x32 product.
__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
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
// Waits until the last products have left the pipe.  Each sum passes through an
// (empty) statement behind the wait, so that nothing reads it earlier.
template <int CF, int RF>
__device__ __forceinline__ void settle_sums(f32x4 (&acc)[CF][RF]) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
    for (int j = 0; j < CF; ++j)
#pragma unroll
        for (int i = 0; i < RF; ++i) asm volatile("" : "+a"(acc[j][i]));
    __builtin_amdgcn_sched_barrier(0);
}
template <typename T>
using Operand = std::conditional_t<std::is_same_v<T, _Float16>, f16x8, bf16x8>;

struct TileArgs {
    const void* rows;     // X [total, depth], or P [total, height]
    const void* cols;     // W [groups, width, depth] / [groups, depth, width], or Q [total, width]
    void*       out;      // [total, width], or [groups, height, width]
    const int*  offsets;  // groups + 1 first rows; null: one group of all rows
    int         groups;
    int         total;    // rows of X, P, Q
    int         height;   // gradient: rows of each group's output
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
template <typename T, int N, bool MAJOR, int THREADS>
struct Operands {
    static constexpr int kPieces = N * kStep / 8 / THREADS;
    static constexpr int kRow    = MAJOR ? N : kStep;  // elements of an LDS row
    static_assert(N * kStep / 8 % THREADS == 0, "whole pieces a thread");
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
    __device__ __forceinline__ void place(const T* first, int row_elements, int valid) {
        ld    = row_elements;
        bound = valid;
        const unsigned odd = static_cast<unsigned>(reinterpret_cast<uintptr_t>(first)) & 2u;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
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
    __device__ __forceinline__ void load(const T* tile, int left, WordPiece (&v)[kPieces]) const {
        const long long rows = MAJOR ? min(left, kStep) : min(bound, N);
        const __amdgpu_buffer_rsrc_t buffer =
            words_buffer(tile, (rows - 1) * ld + (MAJOR ? bound : left));
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            v[i] = load_words<ODD>(buffer, index[i] < left ? at[i] : kAbsent);
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
    T*       out;
    int row0, rows_here, c0, depth, ld_rows, ld_cols;
    long long step_rows, step_cols;
};
template <typename T, int BR, int BC, bool GRAD, bool COLS_MAJOR>
__device__ __forceinline__ bool take_tile(const TileArgs& a, Tile<T>& t) {
    const int col_tiles = (a.width + BC - 1) / BC;
    t.rows = static_cast<const T*>(a.rows);
    t.cols = static_cast<const T*>(a.cols);
    t.out  = static_cast<T*>(a.out);
    int ct;
    if constexpr (GRAD) {
        int rt;
        const int row_tiles = (a.height + BR - 1) / BR;
        if (!tile_of_block(a.groups * row_tiles, col_tiles, rt, ct)) return false;
        const int g = rt / row_tiles;
        t.row0 = (rt % row_tiles) * BR;
        t.rows_here = min(BR, a.height - t.row0);
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
        t.cols += static_cast<long long>(r.group < a.groups ? r.group : 0) * a.width * a.depth +
                  static_cast<long long>(t.c0) * (COLS_MAJOR ? 1 : t.ld_cols);
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
    __device__ __forceinline__ void store(int i) const {
        const int lane = threadIdx.x & 63;
        const int c = c0 + lane % kLanes * 8;
        const int count = min(8, a.width - c);
#pragma unroll
        for (int n = 0; n < 16 / kRows; ++n) {
            const int r = n * kRows + lane / kLanes;
            const float* from = sums + r * kPitch + lane % kLanes * 8;
            float f[8];
            __builtin_memcpy(f, __builtin_assume_aligned(from, 16), 32);
            const uint4 v = piece_from_float<T>(f);
            if (r0 + i * 16 + r < t.rows_here && count > 0) {
                T* p = t.out + static_cast<long long>(r0 + i * 16 + r) * a.width + c;
                if (count == 8) store_piece(p, v);
                else store_part(p, v, count);
            }
        }
    }
};
template <typename T, int RF, int CF>
__device__ __forceinline__ void store_tile(const TileArgs& a, const Tile<T>& t, int r0, int c0,
                                           const f32x4 (&acc)[CF][RF], float* sums) {
    const StoreTile<T, RF, CF> tile{a, t, r0, c0, sums};
    unrolled(std::make_integer_sequence<int, RF>{}, [&](auto at) {
        if (r0 + at.value * 16 < t.rows_here) {
            tile.template put<at.value>(acc);
            tile.store(at.value);
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

// GRAD false: a product (rows operand [s][k], columns operand W as COLS_MAJOR
// says).  GRAD true: a weight gradient (both operands lie along s).
// ADAPT: with the adapters' extension.
//
// The 128 x 128 tile of medium products, and of any sizes and alignment: four waves
// take a quarter each, two buffers of 64 steps.  PIECES: the operands' rows are
// whole 16-byte pieces, which go straight into LDS.  Otherwise they go through
// registers, as the words around each piece, from buffers that end with the operand:
// straight code with eight or sixteen loads under way.  (With a branch a piece for those
// at an edge the compiler waited for each load: 8 groups of 4000 x 4098 over 16384 rows
// 930 us, 810 so; their weights' gradient 1280, 790.  Two workgroups a CU need the
// registers bounded: 1390 with one.)
template <typename T, bool GRAD, bool COLS_MAJOR, bool ADAPT, bool PIECES>
__global__ __launch_bounds__(256, PIECES ? 1 : 2) void tile_product(TileArgs a) {
    constexpr int BR = 128, BC = 128, WC = 2, RF = 4, CF = 4;
    using Rows = Operands<T, BR, GRAD, 256>;
    using Cols = Operands<T, BC, GRAD || COLS_MAJOR, 256>;
    __shared__ __attribute__((aligned(16))) T s_tiles[2 * (BR + BC) * kStep];
    auto rows_at = [&](int it) { return s_tiles + (it & 1) * BR * kStep; };
    auto cols_at = [&](int it) { return s_tiles + (2 * BR + (it & 1) * BC) * kStep; };

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave / WC, wc = wave % WC;
    Tile<T> t;
    if (!take_tile<T, BR, BC, GRAD, COLS_MAJOR>(a, t)) return;

    f32x4 acc[CF][RF];
#pragma unroll
    for (int j = 0; j < CF; ++j)
#pragma unroll
        for (int i = 0; i < RF; ++i) acc[j][i] = f32x4(0.0f);

    const int r0 = wr * RF * 16, c0 = t.c0 + wc * CF * 16;
    const int tiles = (t.depth + kStep - 1) / kStep;
    auto multiply = [&](int it) {
        const T* lr = rows_at(it);
        const T* lc = cols_at(it);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            Operand<T> fr[RF], fc[CF];
#pragma unroll
            for (int i = 0; i < RF; ++i) fr[i] = Rows::read(lr, (wr * RF + i) * 16, half);
#pragma unroll
            for (int j = 0; j < CF; ++j) fc[j] = Cols::read(lc, (wc * CF + j) * 16, half);
#pragma unroll
            for (int j = 0; j < CF; ++j)
#pragma unroll
                for (int i = 0; i < RF; ++i) acc[j][i] = mfma(fc[j], fr[i], acc[j][i]);
        }
    };
    if constexpr (PIECES) {
        Slot<T, GRAD, 64> pr;
        Slot<T, GRAD || COLS_MAJOR, 64> pc;
        pr.place(t.ld_rows, 0, t.rows_here);
        pc.place(t.ld_cols, 0, a.width - t.c0);
        auto load = [&](int it) {
            const u32x4 br = buffer_words(t.rows + it * t.step_rows, 0, 0x7fffffff);
            const u32x4 bc = buffer_words(t.cols + it * t.step_cols, 0, 0x7fffffff);
            const unsigned lr = lds_address(rows_at(it)) + wave * 1024;
            const unsigned lc = lds_address(cols_at(it)) + wave * 1024;
            const int left = t.depth - it * kStep;
            unrolled(std::make_integer_sequence<int, 4>{}, [&](auto i) {
                lds_dma_raw_to<i.value * 4096>(lr);
                asm volatile("s_nop 0");
                lds_dma_raw_x4(br, pr.template offset<i.value>(left));
                lds_dma_raw_to<i.value * 4096>(lc);
                asm volatile("s_nop 0");
                lds_dma_raw_x4(bc, pc.template offset<i.value>(left));
            });
        };
        if (tiles > 0) load(0);
        for (int it = 0; it < tiles; ++it) {
            // every wave's pieces are there, and the other buffer's readers are done
            wait_vmcnt<0>();
            lds_barrier();
            if (it + 1 < tiles) load(it + 1);
            multiply(it);
        }
    } else {
        Rows pr;
        Cols pc;
        pr.place(t.rows, t.ld_rows, t.rows_here);
        pc.place(t.cols, t.ld_cols, a.width - t.c0);
        WordPiece vr[Rows::kPieces], vc[Cols::kPieces];
        auto run = [&](auto odd) {
            auto load = [&](int it) {
                const int left = t.depth - it * kStep;
                pr.template load<odd.value>(t.rows + it * t.step_rows, left, vr);
                pc.template load<odd.value>(t.cols + it * t.step_cols, left, vc);
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
                               static_cast<uintptr_t>(t.ld_rows | t.ld_cols) * 2;
        if (tiles == 0) {
        } else if ((ends & 2) != 0) {
            run(std::true_type{});
        } else {
            run(std::false_type{});
        }
    }
    lds_barrier();  // the operands' LDS is free
    float* sums = reinterpret_cast<float*>(s_tiles) + wave * kStoreFloats<CF>;
    if constexpr (ADAPT) {
        store_adapted<T, RF, CF>(a, t, r0, c0, acc, sums);
    } else {
        store_tile<T, RF, CF>(a, t, r0, c0, acc, sums);
    }
}

// The 64 x 64 tile of products with few tiles and a long contraction: sixteen waves in
// four groups share the contraction, each with its own two buffers, and add up in a fixed
// order.  Any sizes and alignment, as the words around each piece.  Bound by a load's way
// through registers into LDS, about 1 us a turn of 256 steps.  128 rows x 64 x 5120, W
// [k][c], two such tiles or one of 128 x 128: 25 us, 46 with the latter; 1024 x 1024 x
// 4096 24, 43; 823 x 768 x 6787 with adapters 70, 145; a gradient of 256 x 256 from 32768
// rows 136, 287.
template <typename T, bool GRAD, bool COLS_MAJOR, bool ADAPT>
__global__ __launch_bounds__(1024) void tile_product_shared(TileArgs a) {
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

    f32x4 acc[CF][RF];
#pragma unroll
    for (int j = 0; j < CF; ++j)
#pragma unroll
        for (int i = 0; i < RF; ++i) acc[j][i] = f32x4(0.0f);
    const int r0 = wr * RF * 16, c0 = t.c0 + wc * CF * 16;
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
    f32x4(*parts)[4][CF][RF][64] = reinterpret_cast<f32x4(*)[4][CF][RF][64]>(s_tiles);
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
    float* sums = reinterpret_cast<float*>(s_tiles + sizeof(*parts) * GROUPS) + wave * kStoreFloats<CF>;
    if constexpr (ADAPT) {
        store_adapted<T, RF, CF>(a, t, r0, c0, acc, sums);
    } else {
        store_tile<T, RF, CF>(a, t, r0, c0, acc, sums);
    }
}

// The 256 x 256 tile of large products, for operands whose rows are whole 16-byte
// pieces.  Four waves, one a SIMD, take a quarter of 128 x 128 each; 64 steps of
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
//
// 8 groups of 8192 x 4096 over 16384 rows: 887 us a call, 1240 TFLOP/s (the kernel alone
// 869 at best); in one group 783 us at best, 1400, and 808 on average.  The matrix cores
// are busy for 73% of the time, and at that the clock falls to 1.4 - 1.65 GHz (data of
// zeros takes a sixth less time).  That is no limit of the card: a library product of the
// one group keeps them at 89% and takes 740 at best, 789 on average.  What is left lies in
// the two barriers a tile, with their waits for loads, and in the 6 us that a tile costs
// beside its 1.55 us for 64 steps: beginning, first loads and stores.
template <typename T, bool GRAD, bool COLS_MAJOR, bool ADAPT>
__global__ __launch_bounds__(256, 1) void tile_product_wide(TileArgs a) {
    constexpr int BR = 256, BC = 256, RF = 8, CF = 8;
    using RowSlot = Slot<T, GRAD, 128>;
    using ColSlot = Slot<T, GRAD || COLS_MAJOR, 64>;
    using Rows = Operands<T, 128, GRAD, 256>;
    using Cols = Operands<T, 128, GRAD || COLS_MAJOR, 256>;
    extern __shared__ __attribute__((aligned(16))) char s_tiles[];
    constexpr int kSlot = 128 * kStep;  // elements

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave >> 1, wc = wave & 1;
    Tile<T> t;
    if (!take_tile<T, BR, BC, GRAD, COLS_MAJOR>(a, t)) return;

    f32x4 acc[CF][RF];
    const int r0 = wr * RF * 16, c0 = t.c0 + wc * CF * 16;
    const int tiles = (t.depth + kStep - 1) / kStep;
    if (tiles == 0) return zero_tile<BC>(a, t);
    {
        ColSlot cols0, cols1;
        RowSlot low, high;
        cols0.place(t.ld_cols, 0, a.width - t.c0);
        cols1.place(t.ld_cols, 128, a.width - t.c0);
        low.place(t.ld_rows, 0, t.rows_here);
        high.place(t.ld_rows, 64, t.rows_here);
        T* const lds = reinterpret_cast<T*>(s_tiles);
        const unsigned lds0 = lds_address(s_tiles) + wave * 1024;
        auto place_of = [&](int slot) { return lds0 + slot * ColSlot::kBytes; };
        // The tile that is being loaded, as buffers that begin at it, and the
        // contraction steps left there.
        u32x4 rows = buffer_words(t.rows, 0, 0x7fffffff);
        u32x4 cols = buffer_words(t.cols, 0, 0x7fffffff);
        int left = t.depth;
        auto step = [](u32x4& buffer, long long bytes) {
            const unsigned long long at =
                (static_cast<unsigned long long>(buffer[1]) << 32 | buffer[0]) + bytes;
            buffer[0] = static_cast<unsigned>(at);
            buffer[1] = static_cast<unsigned>(at >> 32);
        };
        auto advance = [&] {
            step(rows, t.step_rows * 2);
            step(cols, t.step_cols * 2);
            left -= kStep;
        };
        auto load_slot = [&](const auto& slot, const u32x4& from, unsigned to) {
            unrolled(std::make_integer_sequence<int, 4>{}, [&](auto i) {
                lds_dma_raw_to<i.value * 4096>(to);
                asm volatile("s_nop 0");
                lds_dma_raw_x4(from, slot.template offset<i.value>(left));
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
                if constexpr (m.value % 8 == 6) lds_dma_raw_x4(from, offset);
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
                acc[j][i] = f32x4(0.0f);
                asm volatile("" : "+a"(acc[j][i]));
            }
        wait_vmcnt<24>();  // slots 0, 1, 2
        lds_barrier();
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
            multiply(1, 0, low, rows, place_of(slot), [&](auto m) {
                if constexpr (m.value < 4) read_row(later(3), 0, m.value);
            });
            multiply(0, 1, high, rows, place_of(later(1)), [&](auto m) {
                if constexpr (m.value < 4) read_row(later(3), 1, m.value);
            });
            wait_vmcnt<20>();
            lds_barrier();
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
    float* sums = reinterpret_cast<float*>(s_tiles) + wave * kStoreFloats<CF>;
    if constexpr (ADAPT) {
        store_adapted<T, RF, CF>(a, t, r0, c0, acc, sums);
    } else {
        store_tile<T, RF, CF>(a, t, r0, c0, acc, sums);
    }
}

// Sums of a wave's share of the contraction for CF x 16 columns (rows of `cols`,
// `width` of them from its first) and RF x 16 rows (of `rows`, `rows_here`), all
// with `depth` contiguous elements: wave w of WAVES takes every WAVES-th 64 steps.
// Operands come straight from memory, as the words around each piece; 64 steps' loads
// are under way (with 128, fewer workgroups a CU: 50 rows x 8000 x 1002 15 us, 10 so).
template <typename T, int RF, int CF, int WAVES>
__device__ __forceinline__ void wave_share(const T* rows, int rows_here, const T* cols, int width,
                                           int depth, f32x4 (&acc)[CF][RF]) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int s = lane & 15, q = lane >> 4;
    const unsigned odd_r = static_cast<unsigned>(reinterpret_cast<uintptr_t>(rows)) & 2u;
    const unsigned odd_c = static_cast<unsigned>(reinterpret_cast<uintptr_t>(cols)) & 2u;
    const __amdgpu_buffer_rsrc_t br = words_buffer(rows, static_cast<long long>(rows_here) * depth);
    const __amdgpu_buffer_rsrc_t bc = words_buffer(cols, static_cast<long long>(min(width, CF * 16)) * depth);
    unsigned ar[RF], ac[CF];  // byte offsets of the first piece; rows past the end are zeros
#pragma unroll
    for (int i = 0; i < RF; ++i) {
        const int r = i * 16 + s;
        ar[i] = r < rows_here ? static_cast<unsigned>(r * depth + 8 * q) * 2u + odd_r : kAbsent;
    }
#pragma unroll
    for (int j = 0; j < CF; ++j) {
        const int c = j * 16 + s;
        ac[j] = c < width ? static_cast<unsigned>(c * depth + 8 * q) * 2u + odd_c : kAbsent;
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
                    vc[half][j] = load_words<odd.value>(bc, in ? ac[j] + 2u * at : kAbsent);
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
    if (((odd_r | odd_c) & 2u) != 0 || (depth & 1) != 0) run(std::true_type{});
    else run(std::false_type{});
}

// wave_share for operands whose rows are whole 16-byte pieces (the same sums in the
// same order): a wave's pieces go through a ring of D stages of LDS of its own (no
// barriers).  A load then brings eight rows' whole cache lines; operands read
// straight from memory are 64 bytes of sixteen rows, which the cache serves more
// slowly (8 groups of 4000 columns, 32 rows: 4096 steps 42 us, 4098 47).
//   ring: WAVES x D x (RF + CF) x 2 KB.
template <typename T, int RF, int CF, int WAVES, int D>
__device__ __forceinline__ void ring_share(char* ring, const T* rows, int rows_here, const T* cols,
                                           int width, int depth, f32x4 (&acc)[CF][RF]) {
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
        const int n = 8 * i + (lane >> 3);
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
        const u32x4 br = buffer_words(rows + k, 0, 0x7fffffff);
        unrolled(std::make_integer_sequence<int, 2 * CF>{}, [&](auto i) {
            lds_dma_raw_to<i.value * 1024>(lds0 + slot * kStage);
            asm volatile("s_nop 0");
            lds_dma_raw_x4(bc, in ? at_col[i.value] : kAbsent);
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
template <int RF, int CF, int WAVES>
struct Shares {
    static constexpr int kBytes = WAVES * CF * RF * 1024;
    float (*parts)[CF][RF][64][4];
    __device__ __forceinline__ explicit Shares(char* lds)
        : parts(reinterpret_cast<float (*)[CF][RF][64][4]>(lds)) {}
    __device__ __forceinline__ void put(const f32x4 (&acc)[CF][RF]) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
        for (int j = 0; j < CF; ++j)
#pragma unroll
            for (int i = 0; i < RF; ++i) *reinterpret_cast<f32x4*>(parts[wave][j][i][lane]) = acc[j][i];
    }
    __device__ __forceinline__ float total(int c, int r) const {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            sum += parts[w][c / 16][r / 16][(c % 16) / 4 * 16 + r % 16][c % 4];
        }
        return sum;
    }
};

// h[s, r] = scale_a sum_k X[s, k] A_a[r, k] for RF x 16 rows s and CF x 16 r a
// workgroup, whose waves share the contraction.  h stays in fp32, up to the next whole
// 16 of the rank (zeros behind it).
// The workgroups (x, y, 0 ..) take the adapters among their rows in turn: one each
// where there are as many of them as rows, so that few rows with an adapter each
// still spread over the chip.  Few rows are bound by one workgroup's chain of loads (48
// rows of 4096 with an adapter of rank 16 each: 6.3 us), many by reading the adapters for
// every sixteen rows (8192 rows of 4096, rank 64: 28 us).
//   D: stages of ring_share; 0: wave_share, for rows that are no whole pieces.
template <typename T, int RF, int CF, int WAVES, int D>
__global__ __launch_bounds__(WAVES * 64) void adapter_shrink(TileArgs a, const T* __restrict__ down,
                                                             const float* __restrict__ scale,
                                                             float* __restrict__ h) {
    extern __shared__ __attribute__((aligned(16))) char s_ring[];  // and then the shares
    __shared__ int s_id[RF * 16];
    const int lane = threadIdx.x & 63;
    const int row0 = blockIdx.x * RF * 16;
    const int r0   = blockIdx.y * CF * 16;
    const int rows_here = min(RF * 16, a.total - row0);
    // every wave looks at all the rows' adapters
    int id = lane < rows_here ? a.ids[row0 + lane] : -1;
    if (static_cast<unsigned>(id) >= static_cast<unsigned>(a.adapters)) id = -1;
    if (threadIdx.x < RF * 16) s_id[threadIdx.x] = id;
    unsigned long long left = __ballot(id >= 0);
    int skip = blockIdx.z;
    while (left != 0) {
        const int mine = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        left &= ~__ballot(id == mine);
        if (skip > 0) {
            --skip;
            continue;
        }
        skip = gridDim.z - 1;
        f32x4 acc[CF][RF];
#pragma unroll
        for (int j = 0; j < CF; ++j)
#pragma unroll
            for (int i = 0; i < RF; ++i) acc[j][i] = f32x4(0.0f);
        const T* x = static_cast<const T*>(a.rows) + static_cast<long long>(row0) * a.depth;
        const T* d = down + (static_cast<long long>(mine) * a.rank + r0) * a.depth;
        if (r0 >= a.rank) {
            // only zeros up to rank16
        } else if constexpr (D > 0) {
            ring_share<T, RF, CF, WAVES, D>(s_ring, x, rows_here, d, a.rank - r0, a.depth, acc);
            __syncthreads();
        } else {
            wave_share<T, RF, CF, WAVES>(x, rows_here, d, a.rank - r0, a.depth, acc);
        }
        Shares<RF, CF, WAVES> shares(s_ring);
        shares.put(acc);
        __syncthreads();
        const float f = scale != nullptr ? scale[mine] : 1.0f;
        for (int e = threadIdx.x; e < RF * 16 * CF * 16; e += WAVES * 64) {
            const int s = e / (CF * 16), r = e % (CF * 16);
            if (s_id[s] == mine && r0 + r < a.rank16) {
                h[static_cast<long long>(row0 + s) * a.rank16 + r0 + r] =
                    r0 + r < a.rank ? f * shares.total(r, s) : 0.0f;
            }
        }
        __syncthreads();
    }
}

// Products of few rows, bound by reading the weights (W [c][k]) once: a workgroup
// takes CF x 16 columns and up to RF x 16 rows of a group, its waves share the
// contraction, so that a projection of a few thousand columns still has a workgroup
// a CU.  D: as for adapter_shrink.  64 groups of 2048 x 4096, 256 rows: 168 us, 6.4 TB/s,
// what reads alone reach; 48 rows x 4096 x 4096 with adapters 10.5 us.
template <typename T, int RF, int CF, int WAVES, int D, bool ADAPT>
__global__ __launch_bounds__(WAVES * 64) void few_rows_product(TileArgs a) {
    extern __shared__ __attribute__((aligned(16))) char s_ring[];  // and then the shares
    const int col_tiles = (a.width + CF * 16 - 1) / (CF * 16);
    const RowTile t = find_tile<RF * 16>(a, blockIdx.x / col_tiles);
    if (t.group < 0) return;
    const int c0 = blockIdx.x % col_tiles * CF * 16;
    const int rows_here = t.end - t.first;
    T* out = static_cast<T*>(a.out) + static_cast<long long>(t.first) * a.width;
    f32x4 acc[CF][RF];
#pragma unroll
    for (int j = 0; j < CF; ++j)
#pragma unroll
        for (int i = 0; i < RF; ++i) acc[j][i] = f32x4(0.0f);
    if (t.group < a.groups) {  // rows in no group: zeros
        const T* x = static_cast<const T*>(a.rows) + static_cast<long long>(t.first) * a.depth;
        const T* w = static_cast<const T*>(a.cols) +
                     (static_cast<long long>(t.group) * a.width + c0) * a.depth;
        if constexpr (D > 0) {
            ring_share<T, RF, CF, WAVES, D>(s_ring, x, rows_here, w, a.width - c0, a.depth, acc);
            __syncthreads();
        } else {
            wave_share<T, RF, CF, WAVES>(x, rows_here, w, a.width - c0, a.depth, acc);
        }
    }
    Shares<RF, CF, WAVES> shares(s_ring);
    shares.put(acc);
    __syncthreads();
    const int c = threadIdx.x % (CF * 16);
    if (c0 + c >= a.width) return;
    for (int s = threadIdx.x / (CF * 16); s < rows_here; s += WAVES * 4 / CF) {
        float sum = shares.total(c, s);
        if constexpr (ADAPT) {
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

template <typename T, int RF, int CF, int WAVES, int ROOM, bool ADAPT>
Error launch_few_rows_of(const TileArgs& a, bool pieces, hipStream_t stream, const char* name) {
    const long long row_tiles = a.offsets == nullptr
        ? (a.total + RF * 16 - 1) / (RF * 16)
        : a.total / (RF * 16) + std::min<long long>(a.groups + 2LL, a.total);
    const long long blocks = row_tiles * ((a.width + CF * 16 - 1) / (CF * 16));
    SPMM_TRY(check_threads(blocks, WAVES * 64, name));
    const dim3 grid(static_cast<unsigned>(blocks));
    constexpr int shares = Shares<RF, CF, WAVES>::kBytes;
    if constexpr (CF == 1) {
        if (!pieces) {
            return launch_with_lds<few_rows_product<T, RF, CF, WAVES, 0, ADAPT>>(
                grid, WAVES * 64, shares, stream, name, a);
        }
    }
    constexpr int depth = ring_depth(WAVES, RF + CF, ROOM);
    constexpr int lds = std::max(shares, WAVES * depth * (RF + CF) * 2048);
    return launch_with_lds<few_rows_product<T, RF, CF, WAVES, depth, ADAPT>>(
        grid, WAVES * 64, lds, stream, name, a);
}
// Rows of a group that few_rows_product is launched for: all of one group's, and twice the
// mean of more, so that few of them need a second tile that reads W again.
long long few_rows(const TileArgs& a) {
    const long long groups = a.offsets == nullptr ? 1 : std::min(a.groups, a.total);
    return groups == 1 ? a.total : 2LL * a.total / groups;
}
// How few_rows_product is launched for groups of `rows` rows or so (all are right).
//   Columns: the rows' own reading counts, and 64 columns share it (2048 rows over 64
//     groups of 2048 x 4096: 211 us, 282 with sixteen columns).  For whole pieces only:
//     others, which take longer, are tiles' from there on.
//   Groups: several workgroups a CU hide each other's beginnings and ends (256 rows over
//     64 groups of 2048 x 4096: 167 us with three, 227 with one).
//   Single: a workgroup a CU or so, which has all of the LDS for its loads.
enum class Few { Columns, Groups, Single };
Few few_form(const TileArgs& a, long long rows, bool pieces) {
    const double row_tiles = a.offsets == nullptr ? std::ceil(rows / 64.0) : a.groups;
    if (pieces && rows > 32 && row_tiles * std::ceil(a.width / 64.0) >= 192) return Few::Columns;
    return a.groups > 1 && rows <= 32 ? Few::Groups : Few::Single;
}
template <typename T, bool ADAPT>
Error launch_few_rows(const TileArgs& a, bool pieces, hipStream_t stream, const char* name) {
    constexpr int kAll = 160 * 1024;
    const long long rows = few_rows(a);
    switch (few_form(a, rows, pieces)) {
        case Few::Columns:
            return launch_few_rows_of<T, 4, 4, 4, 80 * 1024, ADAPT>(a, pieces, stream, name);
        case Few::Groups:
            if (rows <= 16) return launch_few_rows_of<T, 1, 1, 4, 54 * 1024, ADAPT>(a, pieces, stream, name);
            return launch_few_rows_of<T, 2, 1, 4, 54 * 1024, ADAPT>(a, pieces, stream, name);
        case Few::Single: break;
    }
    if (rows <= 16) return launch_few_rows_of<T, 1, 1, 8, kAll, ADAPT>(a, pieces, stream, name);
    if (rows <= 32) return launch_few_rows_of<T, 2, 1, 8, kAll, ADAPT>(a, pieces, stream, name);
    if (rows <= 48) return launch_few_rows_of<T, 3, 1, 8, kAll, ADAPT>(a, pieces, stream, name);
    return launch_few_rows_of<T, 4, 1, 8, kAll, ADAPT>(a, pieces, stream, name);
}

template <typename T, int RF, int CF, int WAVES, int ROOM>
Error launch_shrink(const TileArgs& a, bool pieces, const void* down, const float* scale, int turns,
                    hipStream_t stream) {
    // the last columns of h, up to a whole 16, are written (zero) too
    const long long rows = (static_cast<long long>(a.total) + RF * 16 - 1) / (RF * 16);
    SPMM_TRY(check_threads(rows, WAVES * 64, "adapter_shrink"));
    const dim3 grid(static_cast<unsigned>(rows), (a.rank16 + CF * 16 - 1) / (CF * 16), turns);
    const T* d = static_cast<const T*>(down);
    float* h = const_cast<float*>(a.h);
    constexpr int shares = Shares<RF, CF, WAVES>::kBytes;
    if (!pieces) {
        return launch_with_lds<adapter_shrink<T, RF, CF, WAVES, 0>>(
            grid, WAVES * 64, shares, stream, "adapter_shrink", a, d, scale, h);
    }
    constexpr int depth = ring_depth(WAVES, RF + CF, ROOM);
    constexpr int lds = std::max(shares, WAVES * depth * (RF + CF) * 2048);
    return launch_with_lds<adapter_shrink<T, RF, CF, WAVES, depth>>(
        grid, WAVES * 64, lds, stream, "adapter_shrink", a, d, scale, h);
}

// The kernels a product can take: few_rows_product, tile_product through registers
// or with pieces straight into LDS, tile_product_wide, tile_product_shared.
enum class Form { FewRows, Any, Pieces, Wide, Shared };
constexpr int threads_of(Form form) { return form == Form::Shared ? 1024 : 256; }
constexpr int edge_of(Form form) { return form == Form::Wide ? 256 : form == Form::Shared ? 64 : 128; }

// Estimated microseconds of a form for `row_tiles(edge)` x width tiles of `steps`
// steps, from measured rates: 64 steps of a 128 x 128 tile take 0.62 us where a CU has
// one and 0.95 us where it has two (through registers 1 and 1.5 us), of a 256 x 256 tile
// 1.55 us, one a CU, and 256 steps of a 64 x 64 tile 1.1 us, one a CU; `weights` microseconds is what reading the weights takes.
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
    const double two = form == Form::Any ? 1.5 : 0.95, one = form == Form::Any ? 1 : 0.62;
    const double whole = std::floor(tiles / 512), rest = tiles - 512 * whole;
    const double time = whole * (3 + two * rounds) +
                        (rest == 0 ? 0 : 3 + (rest <= 256 ? one : two) * rounds);
    return std::max(time, weights);
}
// The form with the least time; each is right for all sizes that its flag allows.
//   few_rows_product reads weights at 6.3 TB/s, less where the rows' own reading counts;
//     a round of its workgroups takes 2.2 us for 256 steps (64 columns, two a CU) or 1 us
//     for 512 (sixteen, one a CU).
//   Rows that are no whole pieces: 1.1 times as long to read (8 groups of 4000 x 4098,
//     32 rows: 47 us; 64 x 64 tiles 40, 128 x 128 60), twice where they begin between two
//     words (64 groups of 2048 x 4097, 256 rows: 344 us; tiles 222), and 1 us a round for
//     340 steps, 1.3 or 1.65 times, less with fewer rows (20 rows x 4000 x 4097: 17 us,
//     tiles 27).
//   Tiles read W [c][k], a line of each of 128 columns at a time, at 4.1 TB/s, W [k][c]
//     at 5.8 (64 groups of 2048 x 4096, W [c][k]: 256 rows 167 us, tiles 262; 4096 rows
//     257, 285).  Adapters hold tiles up by 6 us, those of 64 x 64 by 5: about what a run of
//     rows with one adapter costs (4000 x 1024 x 1024, rank 16: 5; 701 x 2003 x 1001, rank
//     12: 5; two rounds of 256 x 256, rank 64: 25), less than an adapter a row does (11).
//   64 x 64 tiles: 300 rows x 1024 x 1024 with adapters 14 us, 128 x 128 21; 100 rows x
//     4000 x 4097 30, few_rows_product 43; 12 rows x 1504 x 2057 15, few_rows_product 8.
Form choose_form(const TileArgs& a, bool pieces, bool few_allowed) {
    const double groups = a.offsets == nullptr ? 1 : std::min(a.groups, a.total);
    const double mean = a.total / groups;
    const double weights = 2.0 * groups * a.width * a.depth;
    // groups of all lengths end, on average, in the middle of a tile
    auto row_tiles = [&](int edge) {
        return groups == 1 ? std::ceil(mean / edge) : groups * std::max(1.0, mean / edge + 0.5);
    };
    const bool words = a.depth % 2 == 0 && ((reinterpret_cast<uintptr_t>(a.rows) |
                                             reinterpret_cast<uintptr_t>(a.cols)) & 2) == 0;
    const long long rows = few_rows(a);
    const double tiles64 = groups == 1 ? std::ceil(mean / 64)
                                       : groups * std::max(1.0, mean / 64 + 0.5);
    double few = weights / 6.3e6 * (1 + mean / 160) * (pieces ? 1 : words ? 1.1 : 2);
    switch (few_form(a, rows, pieces)) {
        case Few::Columns:
            few = std::max(few, std::ceil(tiles64 * std::ceil(a.width / 64.0) / 512) *
                                    (2 + 2.2 * std::ceil(a.depth / 256.0)));
            break;
        case Few::Single: {
            const double high  = std::ceil(std::min(rows, 64LL) / 16.0);  // its rows' share of the loads
            const double round = pieces ? 3 + std::ceil(a.depth / 512.0)
                                        : (1 + a.depth / 340.0) * (words ? 1.3 : 1.65) * (high + 2) / 6;
            few = std::max(few, std::ceil(tiles64 * std::ceil(a.width / 16.0) / 256) * round);
            break;
        }
        case Few::Groups: break;
    }
    few += 4;
    const double reading = weights / (few_allowed ? 4.1e6 : 5.8e6);
    auto time = [&](Form f) {
        return tile_time(f, row_tiles, a.width, a.depth, reading) +
               (a.ids == nullptr ? 0 : f == Form::Shared ? 5 : 6);
    };
    Form best = pieces ? Form::Pieces : Form::Any;
    if (pieces && time(Form::Wide) < time(best)) best = Form::Wide;
    if (time(Form::Shared) < time(best)) best = Form::Shared;
    return few_allowed && few <= time(best) ? Form::FewRows : best;
}

// Launches the tile kernel of a form.
template <typename T, bool GRAD, bool COLS_MAJOR, bool ADAPT>
Error launch_tiles(const TileArgs& a, Form form, hipStream_t stream, const char* name) {
    const int edge = edge_of(form);
    // every group may end in a part-filled tile, and so may the rows before and behind them
    const long long row_tiles =
        GRAD ? static_cast<long long>(a.groups) * ((a.height + edge - 1) / edge)
        : a.offsets == nullptr ? (a.total + edge - 1) / edge
                               : a.total / edge + std::min<long long>(a.groups + 2LL, a.total);
    // a whole number of workgroups for each XCD
    const long long blocks = (row_tiles * ((a.width + edge - 1) / edge) + 7) / 8 * 8;
    SPMM_TRY(check_threads(blocks, threads_of(form), name));
    if (form == Form::Wide) {
        return launch_with_lds<tile_product_wide<T, GRAD, COLS_MAJOR, ADAPT>>(
            dim3(static_cast<unsigned>(blocks)), threads_of(Form::Wide), kWideLds, stream, name, a);
    }
    if (form == Form::Shared) {
        return launch_with_lds<tile_product_shared<T, GRAD, COLS_MAJOR, ADAPT>>(
            dim3(static_cast<unsigned>(blocks)), threads_of(Form::Shared), kSharedLds, stream, name, a);
    }
    if (form == Form::Pieces) {
        tile_product<T, GRAD, COLS_MAJOR, ADAPT, true><<<blocks, 256, 0, stream>>>(a);
    } else {
        tile_product<T, GRAD, COLS_MAJOR, ADAPT, false><<<blocks, 256, 0, stream>>>(a);
    }
    SPMM_TRY_HIP(hipGetLastError(), name);
    return Error{};
}

}  // namespace

Error launch_grouped_mm(const void* x, const void* w, ElementType type, const int* offsets,
                        int groups, int total, int width, int depth, bool w_in_rows, void* out,
                        hipStream_t stream) {
    SPMM_TRY(check_product(total, groups, width, depth, "grouped_mm"));
    if (total == 0) return Error{};
    if (x == nullptr || w == nullptr || offsets == nullptr || out == nullptr) {
        return Error{kInvalid, "grouped_mm: null pointer"};
    }
    TileArgs a{};
    a.rows = x;
    a.cols = w;
    a.out = out;
    a.offsets = offsets;
    a.groups = groups;
    a.total = total;
    a.width = width;
    a.depth = depth;
    const bool pieces = depth % 8 == 0 && (!w_in_rows || width % 8 == 0) && aligned16(x) && aligned16(w);
    const Form form = choose_form(a, pieces, !w_in_rows);
    return with_half(type, "grouped_mm", [&](auto zero) {
        using T = decltype(zero);
        if (form == Form::FewRows) return launch_few_rows<T, false>(a, pieces, stream, "grouped_mm");
        return w_in_rows ? launch_tiles<T, false, true, false>(a, form, stream, "grouped_mm")
                         : launch_tiles<T, false, false, false>(a, form, stream, "grouped_mm");
    });
}

Error launch_grouped_outer(const void* p, const void* q, ElementType type, const int* offsets,
                           int groups, int total, int height, int width, void* out,
                           hipStream_t stream) {
    SPMM_TRY(check_product(total, groups, width, height, "grouped_outer"));
    if (offsets == nullptr || out == nullptr || (total > 0 && (p == nullptr || q == nullptr))) {
        return Error{kInvalid, "grouped_outer: null pointer"};
    }
    TileArgs a{};
    a.rows = p;
    a.cols = q;
    a.out = out;
    a.offsets = offsets;
    a.groups = groups;
    a.total = total;
    a.height = height;
    a.width = width;
    const bool pieces = height % 8 == 0 && width % 8 == 0 && aligned16(p) && aligned16(q);
    auto row_tiles = [&](int edge) { return std::ceil(static_cast<double>(height) / edge) * groups; };
    auto time = [&](Form f) {
        return tile_time(f, row_tiles, width, static_cast<double>(total) / groups, 0);
    };
    Form form = !pieces ? Form::Any
                : time(Form::Wide) <= time(Form::Pieces) ? Form::Wide : Form::Pieces;
    if (time(Form::Shared) < time(form)) form = Form::Shared;
    return with_half(type, "grouped_outer", [&](auto zero) {
        using T = decltype(zero);
        return launch_tiles<T, true, true, false>(a, form, stream, "grouped_outer");
    });
}

long long adapter_workspace(long long total, int rank) {
    if (total <= 0 || rank < 1) return 0;
    return total * ((rank + 15LL) / 16 * 16) * static_cast<long long>(sizeof(float));
}

Error launch_adapter_mm(const void* x, const void* w, const void* down, const void* up,
                        const int* ids, const float* scale, ElementType type, int total, int width,
                        int depth, int adapters, int rank, void* out, void* workspace,
                        hipStream_t stream) {
    SPMM_TRY(check_product(total, 1, width, depth, "adapter_mm"));
    if (adapters < 0 || rank < 1) return Error{kInvalid, "adapter_mm: sizes must be positive"};
    if (rank > 1024) return Error{kUnsupported, "adapter_mm: ranks up to 1024"};
    if (total == 0) return Error{};
    if (x == nullptr || w == nullptr || ids == nullptr || out == nullptr || workspace == nullptr ||
        (adapters > 0 && (down == nullptr || up == nullptr))) {
        return Error{kInvalid, "adapter_mm: null pointer"};
    }
    TileArgs a{};
    a.rows = x;
    a.cols = w;
    a.out = out;
    a.groups = 1;
    a.total = total;
    a.width = width;
    a.depth = depth;
    a.ids = ids;
    a.h = static_cast<const float*>(workspace);
    a.b = up;
    a.adapters = adapters;
    a.rank = rank;
    a.rank16 = (rank + 15) / 16 * 16;
    const bool pieces = depth % 8 == 0 && aligned16(x) && aligned16(w);
    a.b_pieces = rank % 8 == 0 && aligned16(up);
    const Form form = choose_form(a, pieces, true);
    return with_half(type, "adapter_mm", [&](auto zero) {
        using T = decltype(zero);
        const bool whole = pieces && aligned16(down);
        if (total <= 512 || (!whole && total <= 2048)) {
            SPMM_TRY((launch_shrink<T, 1, 1, 8, 159 * 1024>(a, whole, down, scale, std::max(1, std::min(16, adapters)), stream)));
        } else {
            SPMM_TRY((launch_shrink<T, 1, 4, 2, 53 * 1024>(a, whole, down, scale, std::max(1, std::min(8, adapters)), stream)));
        }
        if (form == Form::FewRows) return launch_few_rows<T, true>(a, pieces, stream, "adapter_mm");
        return launch_tiles<T, false, false, true>(a, form, stream, "adapter_mm");
    });
}

}  // namespace engine
}  // namespace spmm
