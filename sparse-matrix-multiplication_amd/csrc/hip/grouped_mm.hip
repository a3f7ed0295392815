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

}  // namespace

Error launch_grouped_mm(const void* x, const void* w, ElementType type, const int* offsets,
                        int groups, int total, int width, int depth, bool w_in_rows, void* out,
                        hipStream_t stream) {
    SPMM_TRY(check_product(total, groups, width, depth, "grouped_mm"));
    if (total == 0) return Error{};
    if (x == nullptr || w == nullptr || (offsets == nullptr && groups != 1) || out == nullptr) {
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
    const Form form = choose_form(a, width, pieces, !w_in_rows);
    return with_half(type, "grouped_mm", [&](auto zero) {
        using T = decltype(zero);
        if (form == Form::FewRows) return launch_few_rows<T, Ends::Plain>(a, pieces, stream, "grouped_mm");
        return w_in_rows ? launch_tiles<T, false, true, Ends::Plain>(a, form, stream, "grouped_mm")
                         : launch_tiles<T, false, false, Ends::Plain>(a, form, stream, "grouped_mm");
    });
}

Error launch_grouped_outer(const void* p, const void* q, ElementType type, const int* offsets,
                           int groups, int total, int height, int width, void* out,
                           hipStream_t stream) {
    SPMM_TRY(check_product(total, groups, width, height, "grouped_outer"));
    if ((offsets == nullptr && groups != 1) || out == nullptr || (total > 0 && (p == nullptr || q == nullptr))) {
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
        return launch_tiles<T, true, true, Ends::Plain>(a, form, stream, "grouped_outer");
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
    const Form form = choose_form(a, width, pieces, true);
    return with_half(type, "adapter_mm", [&](auto zero) {
        using T = decltype(zero);
        const bool whole = pieces && aligned16(down);
        if (total <= 512 || (!whole && total <= 2048)) {
            SPMM_TRY((launch_shrink<T, 1, 1, 8, 159 * 1024>(a, whole, down, scale, std::max(1, std::min(16, adapters)), stream)));
        } else {
            SPMM_TRY((launch_shrink<T, 1, 4, 2, 53 * 1024>(a, whole, down, scale, std::max(1, std::min(8, adapters)), stream)));
        }
        if (form == Form::FewRows) return launch_few_rows<T, Ends::Adapters>(a, pieces, stream, "adapter_mm");
        return launch_tiles<T, false, false, Ends::Adapters>(a, form, stream, "adapter_mm");
    });
}

}  // namespace engine
}  // namespace spmm
