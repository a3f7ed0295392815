// Values into eight bits and back:
//
//   pack8          blocks of 32 with a power-of-two scale (eight_bits.h), for activations
//                  that are kept for a backward pass
//   unpack8        the values that they stand for
//   quantize_rows  rows with one fp32 scale, for products in 8-bit integers:
//                  scale = max|x| / 127, q = the integer next to x * (127 / max|x|),
//                  both by reciprocals rounded to fp32; the last product is exact until
//                  it is rounded to an integer
//
// All are bound by memory.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "eight_bits.h"
#include "hip_status.h"

namespace spmm {
namespace engine {
namespace {

using namespace dev;

// A thread takes eight values, four threads a block; blocks never cross rows.
template <typename T>
__global__ __launch_bounds__(256) void pack_blocks(const T* __restrict__ x, unsigned pieces,
                                                   Divisor per_row, int width,
                                                   signed char* __restrict__ values,
                                                   unsigned char* __restrict__ scales) {
    const unsigned p = blockIdx.x * 256u + threadIdx.x;
    if (p >= pieces) return;  // whole fours
    const unsigned row = per_row.quotient(p);
    const int c = static_cast<int>(p - row * per_row.d) * 8;
    const int count = min(8, width - c);
    const long long at = static_cast<long long>(row) * width + c;
    float f[8] = {};
    if (count > 0) load_eight(x + at, count, f);
    const unsigned scale = pack_scale(quad_max(largest_bits(f)));
    if (count > 0) store_bytes(values + at, pack_eight(f, scale), count);
    if (p % 4 == 0) scales[p / 4] = static_cast<unsigned char>(scale);
}

template <typename T>
__global__ __launch_bounds__(256) void unpack_blocks(const signed char* __restrict__ values,
                                                     const unsigned char* __restrict__ scales,
                                                     unsigned pieces, Divisor per_row, int width,
                                                     T* __restrict__ out) {
    const unsigned p = blockIdx.x * 256u + threadIdx.x;
    if (p >= pieces) return;
    const unsigned row = per_row.quotient(p);
    const int c = static_cast<int>(p - row * per_row.d) * 8;
    const int count = min(8, width - c);
    if (count <= 0) return;
    const long long at = static_cast<long long>(row) * width + c;
    float f[8];
    unpack_eight(load_bytes(values + at, count), scales[p / 4], f);
    store_eight(out + at, f, count);
}

// A workgroup takes a row: its first kHeld eights a thread stay in registers between the
// maximum and the rounding, the rest is read again.  16 rows of 8192 2.7 us with sixteen
// waves, 4.2 with four; 8192 rows 31 us again and again (the last cache holds them: 6.5 TB/s),
// 41 between products that take it, 5.0 TB/s; 65536 rows of 256 18, bound by the chain of a
// row's load, maximum and store (four rows a workgroup 17, and 16384 of 2048 17.4 for 16.8).
//   Rows below 2^-100 take that as their largest value: 127 / max (finite down to 2^-121) and
//   max / 127 stay far from fp32's ends, where a product's scales are multiplied one after the
//   other.  Rows below 2^-108 are zeros so.
//   A row with an infinity or a NaN has the scale NaN, which its products become, and zeros.
template <typename T, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void quantize(const T* __restrict__ x, int width, int padded,
                                                       signed char* __restrict__ values,
                                                       float* __restrict__ scales) {
    constexpr int kHeld = WAVES > 4 ? 1 : 4, kStep = WAVES * 64 * 8;
    const T* from = x + static_cast<long long>(blockIdx.x) * width;
    signed char* to = values + static_cast<long long>(blockIdx.x) * padded;
    const int c0 = threadIdx.x * 8;
    float f[kHeld][8] = {};
    unsigned most = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int c = c0 + i * kStep;
        if (c < width) load_eight(from + c, min(8, width - c), f[i]);
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i) most = max(most, largest_bits(f[i]));
    for (int c = c0 + kHeld * kStep; c < width; c += kStep) {
        float g[8];
        load_eight(from + c, min(8, width - c), g);
        most = max(most, largest_bits(g));
    }
    most = group_max<WAVES>(most);
    const bool fine = most < 0x7f800000u;
    const float largest = fmaxf(__uint_as_float(most), 0x1p-100f);
    const float up = fine ? 1.0f / largest * 127.0f : 0.0f;
    auto put = [&](int c, const float (&g)[8]) {
        unsigned q[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = __float_as_uint(fmaf(g[e], up, kRound));
        const u32x2 v = low_bytes(q);
        store_bytes(to + c, fine ? v : u32x2{0u, 0u}, 8);
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int c = c0 + i * kStep;
        if (c < padded) put(c, f[i]);
    }
    for (int c = c0 + kHeld * kStep; c < padded; c += kStep) {
        float g[8] = {};
        if (c < width) load_eight(from + c, min(8, width - c), g);
        put(c, g);
    }
    if (threadIdx.x == 0) {
        scales[blockIdx.x] = !fine ? __builtin_nanf("") : most == 0 ? 0.0f : largest * (1.0f / 127.0f);
    }
}

template <typename F>
Error with_type(ElementType type, F f) {
    switch (type) {
        case ElementType::F32: return f(float{});
        case ElementType::F16: return f(_Float16{});
        case ElementType::BF16: return f(__bf16{});
    }
    return Error{kInvalid, "unknown element type"};
}

Error check_rows(long long rows, int width, const char* name) {
    if (rows < 0 || width < 1) return Error{kInvalid, std::string(name) + ": sizes must be positive"};
    if (width > (1 << 30)) return Error{kUnsupported, std::string(name) + ": rows over 2^30 elements"};
    if (rows > (1LL << 40) / width) {
        return Error{kUnsupported, std::string(name) + ": over 2^40 elements"};
    }
    return Error{};
}

// f(first row, its pieces) for launches of fewer than 2^31 pieces, whole rows each.
template <typename F>
Error by_pieces(long long rows, unsigned per_row, const char* name, F f) {
    const long long most = 0x7fffff00u / per_row;
    for (long long at = 0; at < rows; at += most) {
        f(at, static_cast<unsigned>(std::min(most, rows - at)) * per_row);
        SPMM_TRY_HIP(hipGetLastError(), name);
    }
    return Error{};
}

}  // namespace

Error launch_pack8(const void* x, ElementType type, long long rows, int width, void* values,
                   void* scales, hipStream_t stream) {
    SPMM_TRY(check_rows(rows, width, "pack8"));
    if (rows == 0) return Error{};
    if (x == nullptr || values == nullptr || scales == nullptr) return Error{kInvalid, "pack8: null pointer"};
    const unsigned blocks = (width + kPackBlock - 1) / kPackBlock;
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        return by_pieces(rows, 4 * blocks, "pack8", [&](long long at, unsigned pieces) {
            pack_blocks<T><<<(pieces + 255) / 256, 256, 0, stream>>>(
                static_cast<const T*>(x) + at * width, pieces, Divisor(4 * blocks), width,
                static_cast<signed char*>(values) + at * width,
                static_cast<unsigned char*>(scales) + at * blocks);
        });
    });
}

Error launch_unpack8(const void* values, const void* scales, ElementType type, long long rows,
                     int width, void* out, hipStream_t stream) {
    SPMM_TRY(check_rows(rows, width, "unpack8"));
    if (rows == 0) return Error{};
    if (values == nullptr || scales == nullptr || out == nullptr) {
        return Error{kInvalid, "unpack8: null pointer"};
    }
    const unsigned blocks = (width + kPackBlock - 1) / kPackBlock;
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        return by_pieces(rows, 4 * blocks, "unpack8", [&](long long at, unsigned pieces) {
            unpack_blocks<T><<<(pieces + 255) / 256, 256, 0, stream>>>(
                static_cast<const signed char*>(values) + at * width,
                static_cast<const unsigned char*>(scales) + at * blocks, pieces, Divisor(4 * blocks),
                width, static_cast<T*>(out) + at * width);
        });
    });
}

Error launch_quantize_rows(const void* x, ElementType type, long long rows, int width, void* values,
                           float* scales, hipStream_t stream) {
    SPMM_TRY(check_rows(rows, width, "quantize_rows"));
    if (rows == 0) return Error{};
    if (x == nullptr || values == nullptr || scales == nullptr) {
        return Error{kInvalid, "quantize_rows: null pointer"};
    }
    const int padded = (width + 15) / 16 * 16;
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        // rows of a launch, whose threads HIP counts in 32 bits
        const long long most = kLaunchThreads / 1024;
        for (long long at = 0; at < rows; at += most) {
            const unsigned here = static_cast<unsigned>(std::min(most, rows - at));
            const T* from = static_cast<const T*>(x) + at * width;
            signed char* to = static_cast<signed char*>(values) + at * padded;
            if (width <= 2048) quantize<T, 1><<<here, 64, 0, stream>>>(from, width, padded, to, scales + at);
            else if (here <= 512) quantize<T, 16><<<here, 1024, 0, stream>>>(from, width, padded, to, scales + at);
            else quantize<T, 4><<<here, 256, 0, stream>>>(from, width, padded, to, scales + at);
            SPMM_TRY_HIP(hipGetLastError(), "quantize_rows");
        }
        return Error{};
    });
}

}  // namespace engine
}  // namespace spmm
