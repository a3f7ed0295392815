#pragma once
// Device helpers of the routing and grouped-product kernels: the three element
// types, 16-byte pieces of rows at any 2-byte alignment, and wave reductions.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "amdgcn.h"

namespace spmm {
namespace engine {
namespace dev {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// How many elements a 16-byte piece holds.
template <typename T>
constexpr int kPiece = 16 / static_cast<int>(sizeof(T));

// Sixteen bytes from or to an address that is only aligned for its elements:
// gfx950 runs in unaligned-access mode, so this is one dwordx4 access (split by
// the memory path where it crosses a line, which only costs time).
__device__ __forceinline__ uint4 load_piece(const void* p) {
    uint4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}
// Pieces of 16-bit elements in whole words, from a buffer that begins at the word of an
// operand's first element and ends with the word of its last, so that no other word is
// read; past it are zeros (each word is looked at by itself; no elements: all zeros).
// Sixteen bytes from between two words would take twice the time: those come as the
// words around them and a shift.  Pieces come out of the words later, so that nothing
// waits for a load.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t words_buffer(const void* first, long long elements) {
    const uintptr_t at    = reinterpret_cast<uintptr_t>(first);
    const long long bytes =
        elements > 0 ? (2 * elements + static_cast<long long>(at & 2) + 3) / 4 * 4 : 0;
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(at & ~uintptr_t{2}), 0,
                                             static_cast<int>(bytes < 0x7ffffffc ? bytes : 0x7ffffffc),
                                             kBufWord3);
}
struct WordPiece {
    uint4    words;
    unsigned next;  // ODD only
};
// byte: from the buffer's begin; at or past 2^31 there are zeros.  The next word's 16 is part
// of the offset that the buffer's bounds are checked with; the scalar offset is not.
template <bool ODD>
__device__ __forceinline__ WordPiece load_words(__amdgpu_buffer_rsrc_t buffer, unsigned byte) {
    WordPiece v;
    v.words = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(buffer, byte & ~3u, 0, 0));
    v.next  = ODD ? __builtin_amdgcn_raw_buffer_load_b32(buffer, (byte & ~3u) + 16u, 0, 0) : 0u;
    return v;
}
__device__ __forceinline__ uint4 piece_of(WordPiece v, unsigned byte) {
    const unsigned shift = (byte & 2u) * 8u;
    return uint4{__builtin_amdgcn_alignbit(v.words.y, v.words.x, shift),
                 __builtin_amdgcn_alignbit(v.words.z, v.words.y, shift),
                 __builtin_amdgcn_alignbit(v.words.w, v.words.z, shift),
                 __builtin_amdgcn_alignbit(v.next, v.words.w, shift)};
}
// The first n elements of a piece (any n), zeros behind them.
__device__ __forceinline__ uint4 first_of(uint4 v, int n) {
    auto cut = [&](unsigned w, int e) { return n >= e + 2 ? w : n == e + 1 ? w & 0xffffu : 0u; };
    return uint4{cut(v.x, 0), cut(v.y, 2), cut(v.z, 4), cut(v.w, 6)};
}
__device__ __forceinline__ void store_piece(void* p, uint4 v) { __builtin_memcpy(p, &v, 16); }
// The same for data that the caches are not to keep.
__device__ __forceinline__ void stream_piece(void* p, uint4 v) {
    typedef unsigned words __attribute__((ext_vector_type(4), aligned(2)));
    __builtin_nontemporal_store(words{v.x, v.y, v.z, v.w}, static_cast<words*>(p));
}

// The first `count` elements of a piece (count < kPiece), zeros behind them.
template <typename T>
__device__ __forceinline__ uint4 load_part(const T* p, int count) {
    T e[kPiece<T>];
#pragma unroll
    for (int i = 0; i < kPiece<T>; ++i) e[i] = i < count ? p[i] : static_cast<T>(0.0f);
    return __builtin_bit_cast(uint4, e);
}
template <typename T>
__device__ __forceinline__ void store_part(T* p, uint4 v, int count) {
    T e[kPiece<T>];
    __builtin_memcpy(e, &v, 16);
#pragma unroll
    for (int i = 0; i < kPiece<T>; ++i) {
        if (i < count) p[i] = e[i];
    }
}

template <typename T>
__device__ __forceinline__ void piece_to_float(uint4 v, float (&f)[kPiece<T>]) {
    T e[kPiece<T>];
    __builtin_memcpy(e, &v, 16);
#pragma unroll
    for (int i = 0; i < kPiece<T>; ++i) f[i] = static_cast<float>(e[i]);
}
// Rounds to nearest even: the one rounding of a result held in fp32.
template <typename T>
__device__ __forceinline__ uint4 piece_from_float(const float (&f)[kPiece<T>]) {
    T e[kPiece<T>];
#pragma unroll
    for (int i = 0; i < kPiece<T>; ++i) e[i] = static_cast<T>(f[i]);
    return __builtin_bit_cast(uint4, e);
}

// One step of a wave-wide reduction: the value CTRL's pattern brings to this
// lane, `none` in lanes it brings nothing to.
template <int CTRL>
__device__ __forceinline__ unsigned dpp(unsigned none, unsigned v) {
    return static_cast<unsigned>(__builtin_amdgcn_update_dpp(
        static_cast<int>(none), static_cast<int>(v), CTRL, 0xF, 0xF, false));
}
// Row shifts by 1, 2, 4, 8 gather each row of 16 lanes in its last lane; the
// two broadcasts carry rows 0 and 2 into 1 and 3, then the lower half into the
// upper: lane 63 holds the whole wave's result.
#define SPMM_DPP_STEPS(STEP) STEP(0x111) STEP(0x112) STEP(0x114) STEP(0x118) STEP(0x142) STEP(0x143)

__device__ __forceinline__ unsigned wave_max(unsigned v) {
#define SPMM_STEP(C) { const unsigned o = dpp<C>(0u, v); v = v > o ? v : o; }
    SPMM_DPP_STEPS(SPMM_STEP)
#undef SPMM_STEP
    return static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}
__device__ __forceinline__ float wave_sum(float v) {
#define SPMM_STEP(C) v += __uint_as_float(dpp<C>(0u, __float_as_uint(v)));
    SPMM_DPP_STEPS(SPMM_STEP)
#undef SPMM_STEP
    return __uint_as_float(static_cast<unsigned>(
        __builtin_amdgcn_readlane(static_cast<int>(__float_as_uint(v)), 63)));
}
// Inclusive prefix sums over the lanes of a wave.
__device__ __forceinline__ int wave_prefix(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

}  // namespace dev
}  // namespace engine
}  // namespace spmm
