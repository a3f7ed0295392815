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
// products of the same kernels with twice the columns; in fp16 of rows times a power of two
// each, which is multiplied out of the sums.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "tile_products.h"

namespace spmm {
namespace engine {
namespace {

using namespace dev;

// dg, du and h = act(g) u of a row's columns c .. (count of them, at least one).
template <typename T, bool PACKED>
__device__ __forceinline__ void gradients_of(const T* dh, const void* kept, const unsigned char* kept_scales,
                                             long long row, int c, int count, int width, Act act,
                                             float (&dg)[8], float (&du)[8], float (&h)[8]) {
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
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float value, slope;
        gate_slope(act, g[i], value, slope);
        dg[i] = d[i] * u[i] * slope;
        du[i] = d[i] * value;
        h[i] = value * u[i];
    }
}

// One thread takes eight columns of a row.  Bound by memory: dh, g and u are read and dg, du
// (and h) written once.
//   dg and du are rounded to the operands' type, which the matrix cores take: in bf16 as much
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
    float dg[8], du[8], again[8];
    gradients_of<T, PACKED>(dh, kept, kept_scales, row, c, count, width, act, dg, du, again);
    store_eight(dkept + 2 * row * width + c, dg, count);
    store_eight(dkept + (2 * row + 1) * width + c, du, count);
    if (h != nullptr) store_eight(h + row * width + c, again, count);
}

// Products of two and three fp16 numbers pass fp16's range at either end, as the sums that
// they are terms of need not.  So a row of [dg | du] leaves as its values times 2^-e, and dx
// is multiplied by 2^e in fp32:
//   e = 0 where the row's largest magnitude M lies in [1/2, 2^15), and above that as much as
//     brings it there: the least number that is not lost is below 2^-39 M;
//   e = -16, -32, .. below, whichever brings M into [1/2, 2^15): below 2^-24 M.
// Steps of 16, so that the rows of a group mostly have one e: dW sums over them, and rows of
// another e than the group's largest are multiplied once more before (common_scales).
//   Infinities and NaN do not count for M and stay what they are.
constexpr int kLowestScale = -96, kHighestScale = 112, kNoScale = -112;  // nothing finite but zeros
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<unsigned>(e + 127) << 23); }
__device__ __forceinline__ int row_exponent(unsigned largest) {
    const int a = static_cast<int>(largest >> 23) - 126;  // M < 2^a
    if (largest == 0) return kNoScale;
    return a > 15 ? min(a - 15, kHighestScale) : max(-((15 - a) & ~15), kLowestScale);
}
__device__ __forceinline__ unsigned largest_finite(const float (&f)[8], unsigned most) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned bits = __float_as_uint(f[i]) & 0x7fffffffu;
        if (bits < 0x7f800000u) most = max(most, bits);
    }
    return most;
}

// gated_grad for fp16.  A workgroup takes a row, a thread eight columns of it, which stay in
// registers between the maximum and the rounding.  AGAIN: rows of more, made once for each.
// 20011 rows of 1408: 47 us, 6.0 TB/s (44 in gated_grad, whose threads wait for no maximum).
constexpr int kRowThreads = 1024;
template <bool PACKED, bool AGAIN>
__global__ __launch_bounds__(kRowThreads) void gated_grad_scaled(
    const _Float16* __restrict__ dh, const void* __restrict__ kept,
    const unsigned char* __restrict__ kept_scales, int width, Act act, _Float16* __restrict__ dkept,
    float* __restrict__ row_scales, _Float16* __restrict__ h) {
    __shared__ unsigned s_most[kRowThreads / 64];
    const long long row = blockIdx.x;
    const int c0 = threadIdx.x * 8, step = blockDim.x * 8, lane = threadIdx.x & 63;
    unsigned most = 0;
    auto make = [&](int c, float (&a)[8], float (&b)[8], bool first) {
        const int count = min(8, width - c);
        float again[8];
        gradients_of<_Float16, PACKED>(dh, kept, kept_scales, row, c, count, width, act, a, b, again);
        if (!first) return;
        // what lies behind the row was read as zeros, whose gradients are zeros or, with a
        // block's scale, NaN
        most = largest_finite(b, largest_finite(a, most));
        if (h != nullptr) store_eight(h + row * width + c, again, count);
    };
    float dg[8] = {}, du[8] = {};
    for (int c = c0; c < width; c += step) {
        make(c, dg, du, true);
        if (!AGAIN) break;
    }
    most = wave_max(most);
    if (lane == 0) s_most[threadIdx.x >> 6] = most;
    __syncthreads();
    const int e = row_exponent(wave_max(lane < static_cast<int>(blockDim.x >> 6) ? s_most[lane] : 0u));
    if (threadIdx.x == 0) row_scales[row] = power_of_two(e);
    const float down = power_of_two(-e);
    auto put = [&](int c, float (&a)[8], float (&b)[8]) {
        const int count = min(8, width - c);
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            a[n] *= down;
            b[n] *= down;
        }
        store_eight(dkept + 2 * row * width + c, a, count);
        store_eight(dkept + (2 * row + 1) * width + c, b, count);
    };
    for (int c = c0; c < width; c += step) {
        if (AGAIN) make(c, dg, du, false);
        put(c, dg, du);
        if (!AGAIN) break;
    }
}

// A group's scale, its rows' largest, and the rows of another brought to it.  gridDim.y
// workgroups a group, each of which looks at all of the group's scales (kLoads a thread under
// way) and takes every gridDim.y-th row; rows in no group stay as they are.  4 us where all rows
// have one scale; half of 8192 rows of 11264 brought to the others' 26 us more.
__global__ __launch_bounds__(1024) void common_scales(_Float16* __restrict__ rows, long long elements,
                                                      const int* __restrict__ offsets, int total,
                                                      const float* __restrict__ row_scales,
                                                      float* __restrict__ group_scales) {
    constexpr int kLoads = 8;
    const int g = blockIdx.x;
    auto bound = [&](int i) {
        return offsets == nullptr ? (i == 0 ? 0 : total) : min(max(offsets[i], 0), total);
    };
    const int first = bound(g), end = max(bound(g + 1), first);
    const float none = power_of_two(kNoScale);
    unsigned most = __float_as_uint(none);
    for (long long at = first + static_cast<long long>(threadIdx.x); at < end; at += 1024 * kLoads) {
        float scale[kLoads];
#pragma unroll
        for (int i = 0; i < kLoads; ++i) scale[i] = at + 1024 * i < end ? row_scales[at + 1024 * i] : none;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) most = max(most, __float_as_uint(scale[i]));
    }
    const float scale = __uint_as_float(group_max<16>(most)), down = 1.0f / scale;
    if (blockIdx.y == 0 && threadIdx.x == 0) group_scales[g] = scale;
    // a wave looks at 64 rows' scales at a time; all waves go through those that differ
    const int lane = threadIdx.x & 63, parts = gridDim.y;
    for (long long s0 = first + static_cast<long long>(blockIdx.y); s0 < end; s0 += 64LL * parts) {
        const long long mine = s0 + static_cast<long long>(lane) * parts;
        const float own = mine < end ? row_scales[mine] : none;
        for (unsigned long long left = __ballot(own != scale && own != none); left != 0; left &= left - 1) {
            const int i = __builtin_ctzll(left);
            // never 0, which would make NaN of an infinity
            const float ratio = fmaxf(__shfl(own, i) * down, 0x1p-126f);
            _Float16* row = rows + (s0 + static_cast<long long>(i) * parts) * elements;
            for (long long c = threadIdx.x * 8; c < elements; c += 8192) {
                const int count = static_cast<int>(min(8LL, elements - c));
                float f[8];
                load_eight(row + c, count, f);
#pragma unroll
                for (int n = 0; n < 8; ++n) f[n] *= ratio;
                store_eight(row + c, f, count);
            }
        }
    }
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

namespace {

Error check_grad(const void* dh, const void* kept, int total, int width, Act act, const void* dkept) {
    if (total < 0 || width < 1) return Error{kInvalid, "gated_grad: sizes must be positive"};
    if (!is_act(act)) return Error{kInvalid, "gated_grad: unknown activation"};
    if (width > (1 << 22)) return Error{kUnsupported, "gated_grad: rows over 2^22 elements"};
    if (total > 0 && (dh == nullptr || kept == nullptr || dkept == nullptr)) {
        return Error{kInvalid, "gated_grad: null pointer"};
    }
    return Error{};
}

}  // namespace

Error launch_gated_grad(const void* dh, ElementType type, const void* kept, const void* kept_scales,
                        int total, int width, Act act, void* dkept, void* h, hipStream_t stream) {
    SPMM_TRY(check_grad(dh, kept, total, width, act, dkept));
    if (total == 0) return Error{};
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

Error launch_gated_grad_scaled(const void* dh, const void* kept, const void* kept_scales, int total,
                               int width, Act act, void* dkept, float* row_scales, void* h,
                               hipStream_t stream) {
    SPMM_TRY(check_grad(dh, kept, total, width, act, dkept));
    if (total == 0) return Error{};
    if (row_scales == nullptr) return Error{kInvalid, "gated_grad: null pointer"};
    const int threads = std::min((width + 511) / 512 * 64, kRowThreads);
    // rows of a launch, whose threads HIP counts in 32 bits
    const int most = static_cast<int>(kLaunchThreads / kRowThreads);
    auto launch = [&](auto packed, auto again) {
        constexpr bool kPacked = packed.value;
        for (int at = 0; at < total; at += std::min(most, total - at)) {
            const long long first = static_cast<long long>(at) * width;
            const long long line = 2LL * at * ((width + kPackBlock - 1) / kPackBlock);
            gated_grad_scaled<kPacked, again.value><<<std::min(most, total - at), threads, 0, stream>>>(
                static_cast<const _Float16*>(dh) + first,
                static_cast<const char*>(kept) + 2 * first * (kPacked ? 1 : 2),
                kPacked ? static_cast<const unsigned char*>(kept_scales) + line : nullptr, width, act,
                static_cast<_Float16*>(dkept) + 2 * first, row_scales + at,
                h == nullptr ? nullptr : static_cast<_Float16*>(h) + first);
            SPMM_TRY_HIP(hipGetLastError(), "gated_grad");
        }
        return Error{};
    };
    const bool again = width > 8 * kRowThreads;
    if (kept_scales != nullptr) {
        return again ? launch(std::true_type{}, std::true_type{}) : launch(std::true_type{}, std::false_type{});
    }
    return again ? launch(std::false_type{}, std::true_type{}) : launch(std::false_type{}, std::false_type{});
}

Error launch_common_scales(void* rows, const float* row_scales, const int* offsets, int groups, int total,
                           long long elements, float* group_scales, hipStream_t stream) {
    // groups of a launch, whose threads HIP counts in 32 bits (along x), and workgroups a group:
    // two a CU
    constexpr int most = 1 << 21;
    const int parts = std::max(1, 512 / groups);
    for (int at = 0; at < groups; at += std::min(most, groups - at)) {
        const dim3 grid(std::min(most, groups - at), parts);
        common_scales<<<grid, 1024, 0, stream>>>(static_cast<_Float16*>(rows), elements,
                                                 offsets == nullptr ? nullptr : offsets + at, total, row_scales,
                                                 group_scales + at);
        SPMM_TRY_HIP(hipGetLastError(), "gated_mm_backward");
    }
    return Error{};
}

}  // namespace engine
}  // namespace spmm
