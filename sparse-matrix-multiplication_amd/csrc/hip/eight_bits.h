#pragma once
// Values in eight bits, as blocks of 32 with a power of two for each (MXINT8 of the OCP
// microscaling formats): value = q 2^(scale - 133), q in [-127, 127] and scale a byte.
//   scale: the exponent byte of the block's largest magnitude in fp32, so that this lies
//   in [64, 128) steps; at least 7, which keeps steps normal numbers.  A power of two
//   makes every step of the way exact but the rounding of q itself, and every value that
//   is read back exact in fp16 (from its smallest normal step on) and in bf16.  255: a
//   block with an infinity or a NaN, all of whose values are NaN.
// Eight values are a lane's, four lanes next to each other a block.

#include <hip/hip_runtime.h>

#include "elements.h"
#include "engine.h"

namespace spmm {
namespace engine {
namespace dev {

constexpr int      kPackBlock = 32;
constexpr unsigned kPackLeast = 7u, kPackNone = 255u;

// The largest magnitude as its bits, which order as magnitudes do, infinities and NaN
// above all numbers.
__device__ __forceinline__ unsigned largest_bits(const float (&f)[8]) {
    unsigned most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(f[i]) & 0x7fffffffu);
    return most;
}
// The largest of four lanes 4 n .. 4 n + 3, in each of them.
__device__ __forceinline__ unsigned quad_max(unsigned v) {
    v = max(v, dpp<0xB1>(0u, v));  // lanes 1 0 3 2
    return max(v, dpp<0x4E>(0u, v));  // lanes 2 3 0 1
}
// The largest magnitude's bits over a workgroup of WAVES waves.
template <int WAVES>
__device__ __forceinline__ unsigned group_max(unsigned v) {
    v = wave_max(v);
    if constexpr (WAVES > 1) {
        __shared__ unsigned s_most[WAVES];
        if ((threadIdx.x & 63) == 0) s_most[threadIdx.x >> 6] = v;
        __syncthreads();
        v = s_most[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) v = max(v, s_most[w]);
    }
    return v;
}
__device__ __forceinline__ unsigned pack_scale(unsigned largest) {
    return largest >= 0x7f800000u ? kPackNone : max(largest >> 23, kPackLeast);
}

// The low bytes of eight words.
__device__ __forceinline__ u32x2 low_bytes(const unsigned (&q)[8]) {
    u32x2 v;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const unsigned a = __builtin_amdgcn_perm(q[4 * i + 1], q[4 * i], 0x0c0c0400u);
        const unsigned b = __builtin_amdgcn_perm(q[4 * i + 3], q[4 * i + 2], 0x04000c0cu);
        v[i] = a | b;
    }
    return v;
}
// 1.5 2^23: added to a number below 2^22, it leaves the nearest integer (ties to even) in
// the low bits; in one fused step with a product, which is then rounded only there.
constexpr float kRound = 12582912.0f;

// q of eight values.  Magnitudes above 127.5 steps take 127.
__device__ __forceinline__ u32x2 pack_eight(const float (&f)[8], unsigned scale) {
    const float up = __uint_as_float((260u - scale) << 23);  // 2^(133 - scale)
    unsigned q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float r = fmaf(f[i], up, kRound);
        q[i] = __float_as_uint(__builtin_amdgcn_fmed3f(r, kRound - 127.0f, kRound + 127.0f));
    }
    const u32x2 v = low_bytes(q);
    return scale == kPackNone ? u32x2{0u, 0u} : v;
}
__device__ __forceinline__ void unpack_eight(u32x2 v, unsigned scale, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int q = static_cast<int>(v[i / 4] << (24 - i % 4 * 8)) >> 24;
        f[i] = __builtin_ldexpf(static_cast<float>(q), static_cast<int>(scale) - 133);
        if (scale == kPackNone) f[i] = __builtin_nanf("");
    }
}

// n / d for n below 2^31 by a multiplication: m = ceil(2^(31 + s) / d), 2^s >= d, so that
// m d lies less than 2^s above 2^(31 + s) and the quotient's error below 1 / d.
struct Divisor {
    unsigned d, m, s;
    explicit Divisor(unsigned by) : d(by), s(0) {
        while ((1ull << s) < by) ++s;
        m = static_cast<unsigned>(((1ull << (31 + s)) + by - 1) / by);
    }
    __device__ __forceinline__ unsigned quotient(unsigned n) const {
        return static_cast<unsigned>((static_cast<unsigned long long>(n) * m) >> (31 + s));
    }
};

// Eight bytes from or to any address, and the first `count` of them.
__device__ __forceinline__ u32x2 load_bytes(const void* p, int count) {
    u32x2 v = {0u, 0u};
    if (count >= 8) {
        __builtin_memcpy(&v, p, 8);
        return v;
    }
    const unsigned char* from = static_cast<const unsigned char*>(p);
#pragma unroll
    for (int i = 0; i < 7; ++i) {
        if (i < count) v[i / 4] |= static_cast<unsigned>(from[i]) << (i % 4 * 8);
    }
    return v;
}
__device__ __forceinline__ void store_bytes(void* p, u32x2 v, int count) {
    if (count >= 8) {
        __builtin_memcpy(p, &v, 8);
        return;
    }
    unsigned char* to = static_cast<unsigned char*>(p);
#pragma unroll
    for (int i = 0; i < 7; ++i) {
        if (i < count) to[i] = static_cast<unsigned char>(v[i / 4] >> (i % 4 * 8));
    }
}

// Eight elements from or to any address aligned for them, the first `count` of them (at
// least one); zeros behind those that are read.
template <typename T>
__device__ __forceinline__ void load_eight(const T* p, int count, float (&f)[8]) {
    if constexpr (sizeof(T) == 4) {
        float x[4], y[4];
        piece_to_float<T>(count >= 4 ? load_piece(p) : load_part(p, count), x);
        uint4 high{};
        if (count >= 8) high = load_piece(p + 4);
        else if (count > 4) high = load_part(p + 4, count - 4);
        piece_to_float<T>(high, y);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[i] = x[i];
            f[4 + i] = y[i];
        }
    } else {
        piece_to_float<T>(count >= 8 ? load_piece(p) : load_part(p, count), f);
    }
}
template <typename T>
__device__ __forceinline__ void store_eight(T* p, const float (&f)[8], int count) {
    if constexpr (sizeof(T) == 4) {
        const float x[4] = {f[0], f[1], f[2], f[3]}, y[4] = {f[4], f[5], f[6], f[7]};
        if (count >= 4) store_piece(p, piece_from_float<T>(x));
        else store_part(p, piece_from_float<T>(x), count);
        if (count >= 8) store_piece(p + 4, piece_from_float<T>(y));
        else if (count > 4) store_part(p + 4, piece_from_float<T>(y), count - 4);
    } else {
        const uint4 v = piece_from_float<T>(f);
        if (count >= 8) store_piece(p, v);
        else store_part(p, v, count);
    }
}
// The same to a type that is known at run time, from element `at` on.
__device__ __forceinline__ void store_eight_as(void* out, ElementType type, long long at,
                                               const float (&f)[8], int count) {
    if (type == ElementType::BF16) store_eight(static_cast<__bf16*>(out) + at, f, count);
    else if (type == ElementType::F16) store_eight(static_cast<_Float16*>(out) + at, f, count);
    else store_eight(static_cast<float*>(out) + at, f, count);
}

__device__ __forceinline__ void store_as(void* out, ElementType type, long long at, float f) {
    if (type == ElementType::BF16) static_cast<__bf16*>(out)[at] = static_cast<__bf16>(f);
    else if (type == ElementType::F16) static_cast<_Float16*>(out)[at] = static_cast<_Float16>(f);
    else static_cast<float*>(out)[at] = f;
}

}  // namespace dev
}  // namespace engine
}  // namespace spmm
