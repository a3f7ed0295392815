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
// operand: one block of h a row against the stacked B.  The kernels of tile_products.h do all
// three on matrix cores (v_mfma_f32_16x16x32, fp32 sums).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "tile_products.h"

namespace spmm {
namespace engine {
namespace {

using namespace dev;

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
template <typename T, Ends E>
Error launch_few_rows(const TileArgs& a, bool pieces, hipStream_t stream, const char* name) {
    constexpr int kAll = 160 * 1024;
    const long long rows = few_rows(a);
    switch (few_form(a, rows, pieces)) {
        case Few::Columns:
            return launch_few_rows_of<T, 4, 4, 4, 80 * 1024, E>(a, pieces, stream, name);
        case Few::Groups:
            if (rows <= 16) return launch_few_rows_of<T, 1, 1, 4, 54 * 1024, E>(a, pieces, stream, name);
            return launch_few_rows_of<T, 2, 1, 4, 54 * 1024, E>(a, pieces, stream, name);
        case Few::Single: break;
    }
    if (rows <= 16) return launch_few_rows_of<T, 1, 1, 8, kAll, E>(a, pieces, stream, name);
    if (rows <= 32) return launch_few_rows_of<T, 2, 1, 8, kAll, E>(a, pieces, stream, name);
    if (rows <= 48) return launch_few_rows_of<T, 3, 1, 8, kAll, E>(a, pieces, stream, name);
    return launch_few_rows_of<T, 4, 1, 8, kAll, E>(a, pieces, stream, name);
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
//   Rows of whole words that are no pieces: in tiles as those of pieces, or one of 128 x 128 a
//     CU in a ring (3001 rows in seven groups, 2002 x 1030, W [k][c]: 29 us, 36 in
//     tile_product).  A single group whose rows all know: the ring where there are few tiles of
//     a long contraction (2000 rows x 1024 x 16384, W [k][c]: 107 us, 150 in tile_product).
//   These, and tiles through registers, all add a sum's products in one order; few_rows_product
//     and tile_product_shared have others.  kept: the choice between those three orders is
//     the one of tile_product, so that a product's sums do not change with what else is built.
Form choose_form(const TileArgs& a, bool pieces, bool few_allowed, Lie lie, bool kept,
                 double* least = nullptr) {
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
    Form same = best;  // the fastest of the same order
    if (a.ids == nullptr && lie == Lie::Words) {
        same = time(Form::Pieces) < 0.9 * time(Form::Ring128) ? Form::Pieces : Form::Ring128;
        if (time(Form::Wide) < time(same)) same = Form::Wide;
    }
    if (!kept && a.offsets == nullptr && lie != Lie::Odd) {  // W [k][c]
        // as many rounds of tiles in the ring, which is further ahead of memory
        if (same == Form::Pieces && time(Form::Ring128) < 1.05 * time(same)) same = Form::Ring128;
        if (time(Form::Ring64) < 0.9 * time(same)) same = Form::Ring64;
    }
    const double tiles = time(kept ? best : same);
    Form form = time(Form::Shared) < tiles ? Form::Shared : same;
    if (few_allowed && few <= std::min(tiles, time(Form::Shared))) form = Form::FewRows;
    if (least != nullptr) *least = form == Form::FewRows ? few : time(form);
    return form;
}

}  // namespace

namespace {

// launch_grouped_mm, with the sums in an order that is kept, or free (W [k][c] alone).
// row_scales: null, or what the rows of fp16 sums are multiplied by (W [k][c] alone).
Error product(const void* x, const void* w, ElementType type, const int* offsets, int groups, int total,
              int width, int depth, bool w_in_rows, bool kept, void* out, hipStream_t stream,
              const char* name, const float* row_scales = nullptr) {
    SPMM_TRY(check_product(total, groups, width, depth, name));
    if (total == 0) return Error{};
    if (x == nullptr || w == nullptr || (offsets == nullptr && groups != 1) || out == nullptr) {
        return Error{kInvalid, std::string(name) + ": null pointer"};
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
    a.row_scales = row_scales;
    const bool pieces = depth % 8 == 0 && (!w_in_rows || width % 8 == 0) && aligned16(x) && aligned16(w);
    a.rows_end = static_cast<const char*>(x) + 2LL * total * depth;
    a.cols_end = static_cast<const char*>(w) + 2LL * groups * width * depth;
    const Lie lie = lie_of(a, depth, w_in_rows ? width : depth);
    auto launch = [&](const TileArgs& part, Form form) {
        return with_half(type, name, [&](auto zero) {
            using T = decltype(zero);
            if (form == Form::FewRows) return launch_few_rows<T, Ends::Plain>(part, pieces, stream, name);
            if constexpr (std::is_same_v<T, _Float16>) {
                if (row_scales != nullptr) {
                    return launch_tiles<T, false, true, Ends::Scaled>(part, form, lie, stream, name);
                }
            }
            return w_in_rows ? launch_tiles<T, false, true, Ends::Plain>(part, form, lie, stream, name)
                             : launch_tiles<T, false, false, Ends::Plain>(part, form, lie, stream, name);
        });
    };
    if (!kept && offsets == nullptr && lie != Lie::Odd) {
        const int head = whole_rounds(total, 1, width, [&](int rows, bool wide) {
            TileArgs part = a;
            part.total = rows;
            double time;
            choose_form(part, pieces, !w_in_rows, lie, kept, &time);
            auto tiles = [&](int edge) { return std::ceil(static_cast<double>(rows) / edge); };
            return wide ? tile_time(Form::Wide, tiles, width, depth, 0) : time;
        });
        if (head > 0) {
            SPMM_TRY(launch(rows_alone(a, 0, head, 2), Form::Wide));
            const TileArgs rest = rows_alone(a, head, total - head, 2);
            return launch(rest, choose_form(rest, pieces, !w_in_rows, lie, kept));
        }
    }
    return launch(a, choose_form(a, pieces, !w_in_rows, lie, kept));
}

// launch_grouped_outer, likewise; group_scales: what the groups' fp16 sums are multiplied by.
Error outer(const void* p, const void* q, ElementType type, const int* offsets, int groups, int total,
            int height, int width, bool kept, void* out, hipStream_t stream, const char* name,
            const float* group_scales = nullptr) {
    SPMM_TRY(check_product(total, groups, width, height, name));
    if ((offsets == nullptr && groups != 1) || out == nullptr ||
        (total > 0 && (p == nullptr || q == nullptr))) {
        return Error{kInvalid, std::string(name) + ": null pointer"};
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
    a.group_scales = group_scales;
    const bool pieces = height % 8 == 0 && width % 8 == 0 && aligned16(p) && aligned16(q);
    a.rows_end = static_cast<const char*>(p) + 2LL * total * height;
    a.cols_end = static_cast<const char*>(q) + 2LL * total * width;
    const Lie lie = lie_of(a, height, width);
    // the form with the least time for `rows` of the output's; part: of those that add in one
    // order, so that an element's sum does not hang on the row it is in
    auto choose = [&](int rows, bool part, double* least) {
        auto row_tiles = [&](int edge) { return std::ceil(static_cast<double>(rows) / edge) * groups; };
        auto time = [&](Form f) {
            return tile_time(f, row_tiles, width, static_cast<double>(total) / groups, 0);
        };
        const Form best = !pieces ? Form::Any
                          : time(Form::Wide) <= time(Form::Pieces) ? Form::Wide : Form::Pieces;
        Form same = best;
        if (lie == Lie::Words) {
            same = time(Form::Pieces) < 0.9 * time(Form::Ring128) ? Form::Pieces : Form::Ring128;
            if (time(Form::Wide) < time(same)) same = Form::Wide;
        }
        const Form form = !part && time(Form::Shared) < time(kept ? best : same) ? Form::Shared : same;
        *least = time(form);
        return form;
    };
    auto launch = [&](int from, int upto, Form form) {
        TileArgs part = a;
        part.from = from;
        part.upto = upto;
        return with_half(type, name, [&](auto zero) {
            using T = decltype(zero);
            if constexpr (std::is_same_v<T, _Float16>) {
                if (group_scales != nullptr) {
                    return launch_tiles<T, true, true, Ends::Scaled>(part, form, lie, stream, name);
                }
            }
            return launch_tiles<T, true, true, Ends::Plain>(part, form, lie, stream, name);
        });
    };
    double least;
    Form form = choose(height, false, &least);
    int head = 0;
    if (lie != Lie::Odd && form != Form::Shared) {
        head = whole_rounds(height, groups, width, [&](int rows, bool wide) {
            auto row_tiles = [&](int edge) { return std::ceil(static_cast<double>(rows) / edge) * groups; };
            if (wide) return tile_time(Form::Wide, row_tiles, width, static_cast<double>(total) / groups, 0);
            choose(rows, true, &least);
            return least;
        });
    }
    if (head > 0) {
        SPMM_TRY(launch(0, head, Form::Wide));
        form = choose(height - head, true, &least);
    }
    return launch(head, height, form);
}

}  // namespace

Error launch_grouped_mm(const void* x, const void* w, ElementType type, const int* offsets,
                        int groups, int total, int width, int depth, bool w_in_rows, void* out,
                        hipStream_t stream) {
    return product(x, w, type, offsets, groups, total, width, depth, w_in_rows, true, out, stream,
                   "grouped_mm");
}

Error launch_grouped_outer(const void* p, const void* q, ElementType type, const int* offsets,
                           int groups, int total, int height, int width, void* out,
                           hipStream_t stream) {
    return outer(p, q, type, offsets, groups, total, height, width, true, out, stream, "grouped_outer");
}

Error launch_gated_backward(void* dkept, const float* row_scales, const void* x, const void* w,
                            ElementType type, const int* offsets, int groups, int total, int width,
                            int depth, void* dx, void* dw, float* workspace, hipStream_t stream) {
    const char* name = "gated_mm_backward";
    if (width > 0x3fffffff) return Error{kUnsupported, std::string(name) + ": rows over 2^22 elements"};
    if (dx == nullptr && dw == nullptr) return Error{};
    // all is looked at before anything is launched
    SPMM_TRY(check_product(total, groups, depth, 2 * width, name));
    if (dw != nullptr) SPMM_TRY(check_threads(groups, 256, name));
    if ((offsets == nullptr && groups != 1) ||
        (total > 0 && (dkept == nullptr || (dx != nullptr && w == nullptr) ||
                       (dw != nullptr && (x == nullptr || (row_scales != nullptr && workspace == nullptr)))))) {
        return Error{kInvalid, std::string(name) + ": null pointer"};
    }
    if (dx != nullptr) {
        SPMM_TRY(product(dkept, w, type, offsets, groups, total, depth, 2 * width, true, false, dx,
                         stream, name, row_scales));
    }
    if (dw != nullptr) {
        const float* group_scales = nullptr;
        if (row_scales != nullptr && total > 0) {
            SPMM_TRY(launch_common_scales(dkept, row_scales, offsets, groups, total, 2LL * width, workspace,
                                          stream));
            group_scales = workspace;
        }
        SPMM_TRY(outer(dkept, x, type, offsets, groups, total, 2 * width, depth, false, dw, stream, name,
                       group_scales));
    }
    return Error{};
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
    const Form form = choose_form(a, pieces, true, Lie::Pieces, true);
    return with_half(type, "adapter_mm", [&](auto zero) {
        using T = decltype(zero);
        const bool whole = pieces && aligned16(down);
        if (total <= 512 || (!whole && total <= 2048)) {
            SPMM_TRY((launch_shrink<T, 1, 1, 8, 159 * 1024>(a, whole, down, scale, std::max(1, std::min(16, adapters)), stream)));
        } else {
            SPMM_TRY((launch_shrink<T, 1, 4, 2, 53 * 1024>(a, whole, down, scale, std::max(1, std::min(8, adapters)), stream)));
        }
        if (form == Form::FewRows) return launch_few_rows<T, Ends::Adapters>(a, pieces, stream, "adapter_mm");
        return launch_tiles<T, false, false, Ends::Adapters>(a, form, Lie::Pieces, stream, "adapter_mm");
    });
}

}  // namespace engine
}  // namespace spmm
