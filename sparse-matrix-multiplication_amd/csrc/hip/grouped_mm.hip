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
// operand: one block of h a row against the stacked B.  One tile kernel does all
// three.  A workgroup computes BR rows x BC columns on matrix cores
// (v_mfma_f32_16x16x32, fp32 sums), staging 64 steps of the contraction at a time
// through two LDS buffers.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "amdgcn.h"
#include "elements.h"
#include "engine.h"
#include "hip_status.h"

namespace spmm {
namespace engine {
namespace {

using namespace dev;

constexpr int kStep = 64;  // contraction steps a staged tile holds

// A 16-bit element type's operand of one 16x16x32 product.
__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
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
    const void* h;        // [total, rank32]
    const void* b;        // [adapters, width, rank]
    int         adapters;
    int         rank;
    int         rank32;   // rank rounded up to whole products of 32
};

// The group's rows as the kernels use them: in range and in order whatever the
// offsets hold, so that no value of theirs leads outside the operands.
__device__ __forceinline__ int row_bound(const TileArgs& a, int i) {
    if (a.offsets == nullptr) return i == 0 ? 0 : a.total;
    return min(max(a.offsets[i], 0), a.total);
}

// The row tiles of all groups, counted group by group; past the last group come
// the tiles of the rows in no group (group = groups).  Lane i looks at group i of
// each 64.
struct RowTile {
    int group, first, end;  // rows [first, end), end <= first + BR; group < 0: no such tile
};
__device__ __forceinline__ void group_rows(const TileArgs& a, int g, int& lo, int& hi) {
    lo = hi = 0;
    if (g <= a.groups) {
        lo = row_bound(a, g);
        hi = g < a.groups ? max(row_bound(a, g + 1), lo) : a.total;
    }
}
template <int BR>
__device__ __forceinline__ int count_tiles(const TileArgs& a) {
    if (a.offsets == nullptr) return (a.total + BR - 1) / BR;
    int tiles = 0;
    for (int g0 = 0; g0 <= a.groups; g0 += 64) {
        int lo, hi;
        group_rows(a, g0 + (threadIdx.x & 63), lo, hi);
        tiles += __shfl(wave_prefix((hi - lo + BR - 1) / BR), 63);
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
    int before = 0;
    for (int g0 = 0; g0 <= a.groups; g0 += 64) {
        int lo, hi;
        group_rows(a, g0 + (threadIdx.x & 63), lo, hi);
        const int tiles = (hi - lo + BR - 1) / BR;
        const int upto = before + wave_prefix(tiles);
        const unsigned long long at = __ballot(tile >= upto - tiles && tile < upto);
        if (at != 0) {
            const int l = __builtin_ctzll(at);
            const int first = __shfl(lo + (tile - (upto - tiles)) * BR, l);
            return RowTile{__builtin_amdgcn_readfirstlane(g0 + l),
                           __builtin_amdgcn_readfirstlane(first),
                           __builtin_amdgcn_readfirstlane(min(first + BR, __shfl(hi, l)))};
        }
        before = __shfl(upto, 63);
    }
    return RowTile{-1, 0, 0};
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

// How one operand lies in memory and in LDS.
//   MAJOR false: N rows of the contraction's elements in a row (X, W [c][k]).
//     LDS rows of 64 elements; 16-byte piece p of row n at place p ^ (n & 7), so
//     that the 16 rows of an operand read meet all banks.
//   MAJOR true: the contraction's steps are the rows, N elements each (W [k][c],
//     and both operands of a gradient).  LDS rows of N elements, pieces at place
//     p ^ 2 f(k), f(k) = (k & 3) | ((k >> 3) & 1) << 2: the transposing read of
//     32 lanes takes 32 bytes of rows {0-3, 8-11}, f spreads them over all banks.
template <typename T, int N, bool MAJOR, int THREADS>
struct Operands {
    static constexpr int kPieces = N * kStep / 8 / THREADS;
    static constexpr int kRow    = MAJOR ? N : kStep;  // elements of an LDS row
    static_assert(N * kStep / 8 % THREADS == 0, "whole pieces a thread");
    static_assert(!MAJOR || N >= 128, "the places of a row are 32 bytes x 8");

    int base[kPieces];   // element offset of the piece from the tile's first element
    int index[kPieces];  // its first contraction step inside the tile
    int room[kPieces];   // valid elements of the piece in the other direction's bound (0 - 8)

    // ld: elements between memory rows; bound: valid rows (columns for MAJOR).
    __device__ __forceinline__ void place(int ld, int bound) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int p = i * THREADS + threadIdx.x;
            if constexpr (MAJOR) {
                const int k = p / (N / 8);
                const int f = (k & 3) | ((k >> 3) & 1) << 2;
                const int c = (p % (N / 8)) ^ (f << 1);
                base[i]  = k * ld + c * 8;
                index[i] = k;
                room[i]  = max(0, min(8, bound - c * 8));
            } else {
                const int n = p / 8;
                const int c = (p % 8) ^ (n & 7);
                base[i]  = n * ld + c * 8;
                index[i] = c * 8;
                room[i]  = n < bound ? 8 : 0;
            }
        }
    }
    // Elements of piece i that exist when `left` contraction steps are left.
    __device__ __forceinline__ int count(int i, int left) const {
        if constexpr (MAJOR) return index[i] < left ? room[i] : 0;
        return room[i] == 0 ? 0 : max(0, min(8, left - index[i]));
    }
    __device__ __forceinline__ void load(const T* tile, int left, uint4 (&v)[kPieces]) const {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int n = count(i, left);
            v[i] = n == 8 ? load_piece(tile + base[i]) : n == 0 ? uint4{0, 0, 0, 0}
                                                                : load_part(tile + base[i], n);
        }
    }
    __device__ __forceinline__ void store(T* lds, const uint4 (&v)[kPieces]) const {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            *reinterpret_cast<uint4*>(lds + (i * THREADS + threadIdx.x) * 8) = v[i];
        }
    }
    // Pieces straight into LDS; ld, bound and left are multiples of the piece here, or
    // the piece is past its bound, where the offset past the buffer's end writes zeros.
    // lds: the wave's first place (1 KiB a wave) in LDS.
    __device__ __forceinline__ void dma(u32x4 buffer, unsigned lds, int left, int i) const {
        const unsigned at = index[i] < left && room[i] > 0 ? static_cast<unsigned>(base[i]) * 2u
                                                           : 0x80000000u;
        lds_dma_raw_x4(buffer, lds + i * THREADS * 16, at);
    }
    // Operand of columns n0 .. n0+15, contraction steps 32 half .. +31: lane l holds
    // steps 8 (l >> 4) .. +7 of column l & 15.
    static __device__ __forceinline__ Operand<T> read(const T* lds, int n0, int half) {
        const int lane = threadIdx.x & 63;
        const int q = lane >> 4, s = lane & 15;
        if constexpr (MAJOR) {
            const int k = 32 * half + 8 * q + (s >> 2);
            const int f = (s >> 2) | (q & 1) << 2;
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

// Four consecutive columns of a row from lane values; `count` of them exist.
template <typename T>
__device__ __forceinline__ void store_four(T* p, f32x4 v, int count) {
    T e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = static_cast<T>(v[i]);
    if (count >= 4) {
        __builtin_memcpy(p, e, sizeof(e));
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            if (i < count) p[i] = e[i];
        }
    }
}

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
    int rt, ct;
    if constexpr (GRAD) {
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
        if (!tile_of_block(count_tiles<BR>(a), col_tiles, rt, ct)) return false;
        const RowTile r = find_tile<BR>(a, rt);
        if (r.group < 0) return false;
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

// The adapters' extension of a wave's tile (rows r0 .. of the workgroup's, columns
// c0 ..): the contraction goes on over the adapters of the wave's rows, for each
// that occurs its B against h in the rows that have it.
template <typename T, int RF, int CF>
__device__ __forceinline__ void add_adapters(const TileArgs& a, const Tile<T>& t, int r0, int c0,
                                             f32x4 (&acc)[CF][RF]) {
    const int lane = threadIdx.x & 63;
    const int s = lane & 15, q = lane >> 4;
    const T* h = static_cast<const T*>(a.h);
    const T* b = static_cast<const T*>(a.b);
    int id[RF];
#pragma unroll
    for (int i = 0; i < RF; ++i) {
        const int r = r0 + i * 16 + s;
        id[i] = r < t.rows_here ? a.ids[t.row0 + r] : -1;
        if (static_cast<unsigned>(id[i]) >= static_cast<unsigned>(a.adapters)) id[i] = -1;
    }
#pragma unroll
    for (int i0 = 0; i0 < RF; ++i0) {
        for (;;) {
            const unsigned long long left = __ballot(id[i0] >= 0);
            if (left == 0) break;
            const int mine = __builtin_amdgcn_readlane(id[i0], __builtin_ctzll(left));
            for (int k0 = 0; k0 < a.rank; k0 += 32) {
                const int k = k0 + 8 * q;
                Operand<T> fc[CF];
#pragma unroll
                for (int j = 0; j < CF; ++j) {
                    const int c = c0 + j * 16 + s;
                    const int n = c < a.width ? min(8, a.rank - k) : 0;
                    const T* p = b + (static_cast<long long>(mine) * a.width + c) * a.rank + k;
                    fc[j] = __builtin_bit_cast(Operand<T>, n == 8 ? load_piece(p)
                                                           : n <= 0 ? uint4{0, 0, 0, 0}
                                                                    : load_part(p, n));
                }
#pragma unroll
                for (int i = i0; i < RF; ++i) {
                    if (__ballot(id[i] == mine) == 0) continue;
                    const int r = r0 + i * 16 + s;
                    const uint4 v = id[i] == mine
                        ? load_piece(h + static_cast<long long>(t.row0 + r) * a.rank32 + k)
                        : uint4{0, 0, 0, 0};
                    const Operand<T> fr = __builtin_bit_cast(Operand<T>, v);
                    // A lane's sums are its own row's: other rows keep theirs,
                    // whatever (infinities, NaN) this adapter's B holds.
#pragma unroll
                    for (int j = 0; j < CF; ++j) {
                        const f32x4 next = mfma(fc[j], fr, acc[j][i]);
                        acc[j][i] = id[i] == mine ? next : acc[j][i];
                    }
                }
            }
#pragma unroll
            for (int i = i0; i < RF; ++i) id[i] = id[i] == mine ? -1 : id[i];
        }
    }
}

template <typename T, int RF, int CF>
__device__ __forceinline__ void store_tile(const TileArgs& a, const Tile<T>& t, int r0, int c0,
                                           const f32x4 (&acc)[CF][RF]) {
    const int lane = threadIdx.x & 63;
    const int s = lane & 15, q = lane >> 4;
#pragma unroll
    for (int i = 0; i < RF; ++i) {
        const int r = r0 + i * 16 + s;
        if (r >= t.rows_here) continue;
#pragma unroll
        for (int j = 0; j < CF; ++j) {
            const int c = c0 + j * 16 + 4 * q;
            store_four(t.out + static_cast<long long>(r) * a.width + c, acc[j][i], a.width - c);
        }
    }
}

// GRAD false: a product (rows operand [s][k], columns operand W as COLS_MAJOR
// says).  GRAD true: a weight gradient (both operands lie along s).
// ADAPT: with the adapters' extension.
//
// tile_product takes any sizes and alignment: pieces go through registers, those
// at an edge element by element.
template <typename T, int BR, int BC, int WR, int WC, bool GRAD, bool COLS_MAJOR, bool ADAPT>
__global__ __launch_bounds__(WR * WC * 64) void tile_product(TileArgs a) {
    constexpr int THREADS = WR * WC * 64;
    constexpr int RF = BR / WR / 16, CF = BC / WC / 16;  // 16 x 16 tiles a wave
    using Rows = Operands<T, BR, GRAD, THREADS>;
    using Cols = Operands<T, BC, GRAD || COLS_MAJOR, THREADS>;
    __shared__ __attribute__((aligned(16))) T s_rows[2][BR * kStep];
    __shared__ __attribute__((aligned(16))) T s_cols[2][BC * kStep];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave / WC, wc = wave % WC;
    Tile<T> t;
    if (!take_tile<T, BR, BC, GRAD, COLS_MAJOR>(a, t)) return;

    f32x4 acc[CF][RF];
#pragma unroll
    for (int j = 0; j < CF; ++j)
#pragma unroll
        for (int i = 0; i < RF; ++i) acc[j][i] = f32x4(0.0f);

    Rows pr;
    Cols pc;
    pr.place(t.ld_rows, t.rows_here);
    pc.place(t.ld_cols, a.width - t.c0);
    const int tiles = (t.depth + kStep - 1) / kStep;
    uint4 vr[Rows::kPieces], vc[Cols::kPieces];
    if (tiles > 0) {
        pr.load(t.rows, t.depth, vr);
        pc.load(t.cols, t.depth, vc);
        pr.store(s_rows[0], vr);
        pc.store(s_cols[0], vc);
    }
    for (int it = 0; it < tiles; ++it) {
        // the tile is written, and the other buffer's readers are done
        __syncthreads();
        const bool more = it + 1 < tiles;
        if (more) {
            const int left = t.depth - (it + 1) * kStep;
            pr.load(t.rows + (it + 1) * t.step_rows, left, vr);
            pc.load(t.cols + (it + 1) * t.step_cols, left, vc);
        }
        const T* lr = s_rows[it & 1];
        const T* lc = s_cols[it & 1];
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
        if (more) {
            pr.store(s_rows[(it + 1) & 1], vr);
            pc.store(s_cols[(it + 1) & 1], vc);
        }
    }
    if constexpr (ADAPT) add_adapters<T, RF, CF>(a, t, wr * RF * 16, t.c0 + wc * CF * 16, acc);
    store_tile<T, RF, CF>(a, t, wr * RF * 16, t.c0 + wc * CF * 16, acc);
}

// The 256 x 256 tile of large products, for operands whose rows are whole 16-byte
// pieces: pieces go straight into LDS, and two groups of four waves (one a SIMD
// each) take turns.  While one group reads a quarter of a staged tile's operands,
// the other multiplies the quarter it has read; a barrier swaps them.  A quarter
// is 16 products of 16x16x32 a wave (256 cycles), against 4 to 8 operand reads a
// wave for four waves (128 to 256 cycles of the LDS).
//   Buffer it & 1 is overwritten only in iteration it + 1: a group gets there
//   after the barrier that follows the other group's last reads of it.
//   A tile's loads are issued in the first two quarters of the tile before and
//   waited for (each wave its own) in the last quarter before the barrier, after
//   which either group may read it.
template <typename T, bool GRAD, bool COLS_MAJOR, bool ADAPT>
__global__ __launch_bounds__(512) void tile_product_wide(TileArgs a) {
    constexpr int BR = 256, BC = 256, THREADS = 512, RF = 8, CF = 4;
    using Rows = Operands<T, BR, GRAD, THREADS>;
    using Cols = Operands<T, BC, GRAD || COLS_MAJOR, THREADS>;
    extern __shared__ __attribute__((aligned(16))) char s_tiles[];
    constexpr int kTile = BR * kStep;  // elements of an operand's tile

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave >> 2, wc = wave & 3;
    Tile<T> t;
    if (!take_tile<T, BR, BC, GRAD, COLS_MAJOR>(a, t)) return;

    f32x4 acc[CF][RF];
#pragma unroll
    for (int j = 0; j < CF; ++j)
#pragma unroll
        for (int i = 0; i < RF; ++i) acc[j][i] = f32x4(0.0f);

    Rows pr;
    Cols pc;
    pr.place(t.ld_rows, t.rows_here);
    pc.place(t.ld_cols, a.width - t.c0);
    const int tiles = (t.depth + kStep - 1) / kStep;
    T* const lds = reinterpret_cast<T*>(s_tiles);
    const unsigned lds0 = lds_address(s_tiles) + wave * 1024;
    auto load_rows = [&](int it) {
        const u32x4 buffer = buffer_words(t.rows + it * t.step_rows, 0, 0x7fffffff);
#pragma unroll
        for (int i = 0; i < Rows::kPieces; ++i) {
            pr.dma(buffer, lds0 + (it & 1) * 4 * kTile, t.depth - it * kStep, i);
        }
    };
    auto load_cols = [&](int it) {
        const u32x4 buffer = buffer_words(t.cols + it * t.step_cols, 0, 0x7fffffff);
#pragma unroll
        for (int i = 0; i < Cols::kPieces; ++i) {
            pc.dma(buffer, lds0 + (it & 1) * 4 * kTile + 2 * kTile, t.depth - it * kStep, i);
        }
    };
    if (tiles > 0) {
        load_rows(0);
        load_cols(0);
        wait_vmcnt<0>();
        lds_barrier();
        if (wr == 1) lds_barrier();
    }
    for (int it = 0; it < tiles; ++it) {
        const T* lr = lds + (it & 1) * 2 * kTile;
        const T* lc = lr + kTile;
        Operand<T> fc[CF], fr[RF / 2];
#pragma unroll
        for (int part = 0; part < 4; ++part) {
            const int half = part >> 1, i0 = (part & 1) * (RF / 2);
            if ((part & 1) == 0) {
#pragma unroll
                for (int j = 0; j < CF; ++j) fc[j] = Cols::read(lc, (wc * CF + j) * 16, half);
            }
#pragma unroll
            for (int i = 0; i < RF / 2; ++i) {
                fr[i] = Rows::read(lr, (wr * RF + i0 + i) * 16, half);
            }
            if (it + 1 < tiles) {
                if (part == 0) load_rows(it + 1);
                if (part == 1) load_cols(it + 1);
            }
            if (part == 3) wait_vmcnt<0>();
            __builtin_amdgcn_sched_barrier(0);
            lds_barrier();
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int j = 0; j < CF; ++j)
#pragma unroll
                for (int i = 0; i < RF / 2; ++i) acc[j][i0 + i] = mfma(fc[j], fr[i], acc[j][i0 + i]);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            lds_barrier();
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (tiles > 0 && wr == 0) lds_barrier();  // the other group's last one
    if constexpr (ADAPT) add_adapters<T, RF, CF>(a, t, wr * RF * 16, t.c0 + wc * CF * 16, acc);
    store_tile<T, RF, CF>(a, t, wr * RF * 16, t.c0 + wc * CF * 16, acc);
}

// h[s, r] = scale_a sum_k X[s, k] A_a[r, k] for 16 rows s and 16 r a workgroup:
// four waves share the contraction, every adapter among the rows takes a turn.
// h is rounded to the operands' type: it feeds matrix cores again, and its
// rounding adds less to the result than the result's own (the adapter's part of
// an output averages `rank` such roundings).
template <typename T>
__global__ __launch_bounds__(256) void adapter_shrink(TileArgs a, const T* __restrict__ down,
                                                      const float* __restrict__ scale,
                                                      T* __restrict__ h) {
    __shared__ f32x4 s_part[4][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int s = lane & 15, q = lane >> 4;
    const int row = blockIdx.x * 16 + s;
    const int r0  = blockIdx.y * 16;
    int id = row < a.total ? a.ids[row] : -1;
    if (static_cast<unsigned>(id) >= static_cast<unsigned>(a.adapters)) id = -1;
    const T* x = static_cast<const T*>(a.rows) + static_cast<long long>(row) * a.depth;
    int left_id = id;
    for (;;) {
        const unsigned long long left = __ballot(left_id >= 0);
        if (left == 0) break;
        const int mine = __builtin_amdgcn_readlane(left_id, __builtin_ctzll(left));
        const T* d = down + (static_cast<long long>(mine) * a.rank + r0 + s) * a.depth;
        f32x4 acc = f32x4(0.0f);
        for (int k = wave * 32 + 8 * q; k < (a.depth + 31) / 32 * 32 + 8 * q; k += 128) {
            const int n = min(8, a.depth - k);
            uint4 vx = {0, 0, 0, 0}, va = {0, 0, 0, 0};
            if (n > 0) {
                if (id == mine) vx = n == 8 ? load_piece(x + k) : load_part(x + k, n);
                if (r0 + s < a.rank) va = n == 8 ? load_piece(d + k) : load_part(d + k, n);
            }
            acc = mfma(__builtin_bit_cast(Operand<T>, va), __builtin_bit_cast(Operand<T>, vx), acc);
        }
        s_part[wave][lane] = acc;
        __syncthreads();
        if (wave == 0 && id == mine) {
            const float f = scale != nullptr ? scale[mine] : 1.0f;
            T e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                e[i] = static_cast<T>(f * ((s_part[0][lane][i] + s_part[1][lane][i]) +
                                           (s_part[2][lane][i] + s_part[3][lane][i])));
            }
            __builtin_memcpy(h + static_cast<long long>(row) * a.rank32 + r0 + 4 * q, e, 8);
        }
        __syncthreads();
        left_id = left_id == mine ? -1 : left_id;
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
    return Error{};
}

template <typename F>
Error with_half(ElementType type, const char* name, F f) {
    if (type == ElementType::F16) return f(_Float16{});
    if (type == ElementType::BF16) return f(__bf16{});
    return Error{kUnsupported, std::string(name) + ": fp16 or bf16 operands (matrix cores)"};
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

constexpr size_t kWideLds = 2 * 2 * 256 * kStep * 2;  // two buffers of two operands

// Launches the tile kernel for a: the wide one where the operands' rows are whole
// pieces and `wide` says that its tiles fill.
template <typename T, bool GRAD, bool COLS_MAJOR, bool ADAPT>
Error launch_tiles(const TileArgs& a, bool wide, hipStream_t stream, const char* name) {
    const int edge = wide ? 256 : 128;
    // every group may end in a part-filled tile, and so may the rows in no group
    const long long row_tiles =
        GRAD ? static_cast<long long>(a.groups) * ((a.height + edge - 1) / edge)
        : a.offsets == nullptr ? (a.total + edge - 1) / edge
                               : a.total / edge + std::min<long long>(a.groups + 1LL, a.total);
    // a whole number of workgroups for each XCD
    const long long blocks = (row_tiles * ((a.width + edge - 1) / edge) + 7) / 8 * 8;
    if (blocks > 0x7fffffffLL) return Error{kUnsupported, std::string(name) + ": too many tiles"};
    if (wide) {
        static const hipError_t grown = hipFuncSetAttribute(
            reinterpret_cast<const void*>(tile_product_wide<T, GRAD, COLS_MAJOR, ADAPT>),
            hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kWideLds));
        SPMM_TRY_HIP(grown, name);
        tile_product_wide<T, GRAD, COLS_MAJOR, ADAPT><<<blocks, 512, kWideLds, stream>>>(a);
    } else {
        tile_product<T, 128, 128, 2, 2, GRAD, COLS_MAJOR, ADAPT><<<blocks, 256, 0, stream>>>(a);
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
    const bool wide = pieces && total >= 192LL * groups && width >= 192;
    return with_half(type, "grouped_mm", [&](auto zero) {
        using T = decltype(zero);
        return w_in_rows ? launch_tiles<T, false, true, false>(a, wide, stream, "grouped_mm")
                         : launch_tiles<T, false, false, false>(a, wide, stream, "grouped_mm");
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
    const bool wide = pieces && height >= 192 && width >= 192;
    return with_half(type, "grouped_outer", [&](auto zero) {
        using T = decltype(zero);
        return launch_tiles<T, true, true, false>(a, wide, stream, "grouped_outer");
    });
}

long long adapter_workspace(long long total, int rank) {
    if (total <= 0 || rank < 1) return 0;
    return total * ((rank + 31LL) / 32 * 32) * 2;
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
    a.h = workspace;
    a.b = up;
    a.adapters = adapters;
    a.rank = rank;
    a.rank32 = (rank + 31) / 32 * 32;
    const bool wide = depth % 8 == 0 && aligned16(x) && aligned16(w) && total >= 192 && width >= 192;
    return with_half(type, "adapter_mm", [&](auto zero) {
        using T = decltype(zero);
        // whole products of 32: the second half of h's columns is written (zero) too
        adapter_shrink<T><<<dim3((total + 15) / 16, a.rank32 / 16), 256, 0, stream>>>(
            a, static_cast<const T*>(down), scale, static_cast<T*>(workspace));
        SPMM_TRY_HIP(hipGetLastError(), "adapter_shrink");
        return launch_tiles<T, false, false, true>(a, wide, stream, "adapter_mm");
    });
}

}  // namespace engine
}  // namespace spmm
