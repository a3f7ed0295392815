// Gated products: both projections of a feed-forward block, the activation and the product
// in one kernel, and the elementwise part of their gradients:
//
//   forward    g = x Wg^T, u = x Wu^T, h = act(g) * u
//   backward   dg = dh * u * act'(g), du = dh * act(g), from g and u as they were kept
//
// The projections are the tile kernels' products whose column tiles take half of their
// columns from either weights, so that a wave holds g and u of the same places in its sums
// and nothing but h (and what is kept) is written.  g and u are fp32 sums until h is
// rounded.  dx = [dg | du] [Wg; Wu] and the weights' gradients [dg | du]^T x are then
// products of the same kernels with twice the columns.

#include <hip/hip_runtime.h>

#include "tile_products.h"

namespace spmm {
namespace engine {
namespace {

using namespace dev;

// One thread takes eight columns of a row.  Bound by memory: dh, g and u are read and dg, du
// (and h) written once.
//   dg and du are rounded to the operands' type, which the matrix cores take: as much
//   again as the rounding of the results that they are summed up to.
template <typename T, bool PACKED>
__global__ __launch_bounds__(256) void gated_grad(const T* __restrict__ dh, const void* __restrict__ kept,
                                                  const unsigned char* __restrict__ kept_scales,
                                                  unsigned pieces, Divisor per_row, int width, Act act,
                                                  T* __restrict__ dkept, T* __restrict__ h) {
    const unsigned p = blockIdx.x * 256u + threadIdx.x;
    if (p >= pieces) return;
    const long long row = per_row.quotient(p);
    const int c = static_cast<int>(p - static_cast<unsigned>(row) * per_row.d) * 8;
    const int count = min(8, width - c);
    const long long gate = 2 * row * width + c, other = gate + width;
    float d[8], g[8], u[8];
    load_eight(dh + row * width + c, count, d);
    if constexpr (PACKED) {
        const signed char* q = static_cast<const signed char*>(kept);
        const long long blocks = (width + kPackBlock - 1) / kPackBlock;
        const unsigned char* scale = kept_scales + 2 * row * blocks + c / kPackBlock;
        unpack_eight(load_bytes(q + gate, count), scale[0], g);
        unpack_eight(load_bytes(q + other, count), scale[blocks], u);
    } else {
        load_eight(static_cast<const T*>(kept) + gate, count, g);
        load_eight(static_cast<const T*>(kept) + other, count, u);
    }
    float dg[8], du[8], again[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float value, slope;
        gate_slope(act, g[i], value, slope);
        dg[i] = d[i] * u[i] * slope;
        du[i] = d[i] * value;
        again[i] = value * u[i];
    }
    store_eight(dkept + gate, dg, count);
    store_eight(dkept + other, du, count);
    if (h != nullptr) store_eight(h + row * width + c, again, count);
}

bool is_act(Act act) { return act >= Act::Silu && act <= Act::GeluTanh; }

}  // namespace

Error launch_gated_mm(const void* x, const void* w, ElementType type, const int* offsets, int groups,
                      int total, int width, int depth, Act act, void* out, void* kept,
                      void* kept_scales, hipStream_t stream) {
    SPMM_TRY(check_product(total, groups, width, depth, "gated_mm"));
    if (!is_act(act)) return Error{kInvalid, "gated_mm: unknown activation"};
    if (total == 0) return Error{};
    if (x == nullptr || w == nullptr || (offsets == nullptr && groups != 1) || out == nullptr ||
        (kept_scales != nullptr && kept == nullptr)) {
        return Error{kInvalid, "gated_mm: null pointer"};
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
    a.act = act;
    a.kept = kept;
    a.kept_scales = static_cast<unsigned char*>(kept_scales);
    a.rows_end = static_cast<const char*>(x) + 2LL * total * depth;
    a.cols_end = static_cast<const char*>(w) + 4LL * groups * width * depth;
    const Lie lie = lie_of(a, depth, depth);
    return with_half(type, "gated_mm", [&](auto zero) {
        return launch_finished<decltype(zero), Ends::Gated>(a, lie, stream, "gated_mm");
    });
}

Error launch_gated_int8_mm(const void* x, const float* x_scales, const void* w, const float* w_scales,
                           const int* offsets, int groups, int total, int width, int depth, Act act,
                           ElementType out_type, void* out, hipStream_t stream) {
    if (!is_act(act)) return Error{kInvalid, "gated_int8_mm: unknown activation"};
    TileArgs a{};
    SPMM_TRY(int8_args(x, x_scales, w, w_scales, offsets, groups, total, width, depth, out_type, out,
                       "gated_int8_mm", a));
    if (total == 0) return Error{};
    a.act = act;
    return launch_finished<Int8Pair, Ends::Gated>(a, Lie::Pieces, stream, "gated_int8_mm");
}

Error launch_gated_grad(const void* dh, ElementType type, const void* kept, const void* kept_scales,
                        int total, int width, Act act, void* dkept, void* h, hipStream_t stream) {
    if (total < 0 || width < 1) return Error{kInvalid, "gated_grad: sizes must be positive"};
    if (!is_act(act)) return Error{kInvalid, "gated_grad: unknown activation"};
    if (width > (1 << 22)) return Error{kUnsupported, "gated_grad: rows over 2^22 elements"};
    if (total == 0) return Error{};
    if (dh == nullptr || kept == nullptr || dkept == nullptr) {
        return Error{kInvalid, "gated_grad: null pointer"};
    }
    const int per_row = (width + 7) / 8;
    return with_half(type, "gated_grad", [&](auto zero) {
        using T = decltype(zero);
        // rows of one launch: their pieces stay below 2^31
        const int most = 0x7fffff00 / per_row;
        for (int at = 0; at < total; at += std::min(most, total - at)) {
            const unsigned pieces = static_cast<unsigned>(std::min(most, total - at)) * per_row;
            const unsigned blocks = (pieces + 255) / 256;
            const long long first = static_cast<long long>(at) * width;
            const T* d = static_cast<const T*>(dh) + first;
            T* dk = static_cast<T*>(dkept) + 2 * first;
            T* again = h == nullptr ? nullptr : static_cast<T*>(h) + first;
            if (kept_scales != nullptr) {
                const long long line = 2LL * at * ((width + kPackBlock - 1) / kPackBlock);
                gated_grad<T, true><<<blocks, 256, 0, stream>>>(
                    d, static_cast<const signed char*>(kept) + 2 * first,
                    static_cast<const unsigned char*>(kept_scales) + line, pieces, Divisor(per_row),
                    width, act, dk, again);
            } else {
                gated_grad<T, false><<<blocks, 256, 0, stream>>>(
                    d, static_cast<const T*>(kept) + 2 * first, nullptr, pieces, Divisor(per_row), width,
                    act, dk, again);
            }
            SPMM_TRY_HIP(hipGetLastError(), "gated_grad");
        }
        return Error{};
    });
}

}  // namespace engine
}  // namespace spmm
