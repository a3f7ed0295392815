// Tokens into expert order and back: products of the routing matrix (k entries
// a token, slots[t, j] the row in expert order or -1) with dense rows.
//
//   dispatch            xs[slot(t,j)] = x[t]; rows behind the last group are 0
//   gather              y[t]  = sum_j w[t,j] ys[slot(t,j)]    combine; w = 1: dispatch's gradient
//   combine_backward    dys[slot(t,j)] = w[t,j] dy[t],  dw[t,j] = <dy[t], ys[slot(t,j)]>
//
// All of it is memory traffic.  A token's row is read once and written to its k
// slots (or the other way round), in 16-byte pieces, by one wave, or by a
// workgroup where there are too few tokens to fill the chip with waves.  Sums
// run over j in order, in fp32, and are rounded once.  8192 tokens x 8 x 4096 bf16:
// dispatch 105 us (5.7 TB/s; a copy reaches 5.2), combine 130 (4.6), combine_backward 249
// (4.6).  5003 x 4 x 2050 fp32, whose rows start inside lines: combine_backward 77 us,
// dispatch's gradient 57 (4.9 and 3.6 TB/s; four 16-byte loads a lane are under way, and
// the next columns' begin when they are used).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "elements.h"
#include "engine.h"
#include "hip_status.h"

namespace spmm {
namespace engine {
namespace {

using namespace dev;

struct Rows {
    int  tokens, k, features;
    int  total;  // slots, of all launches' tokens
    bool clear;  // this launch writes the rows without an entry
};

// A slot as a scalar: the same for a whole wave.
__device__ __forceinline__ int slot_of(const int* slots, long long i) {
    return __builtin_amdgcn_readfirstlane(slots[i]);
}

// Zeros in the rows that no entry has, a row a workgroup at a time.
template <typename T>
__device__ __forceinline__ void zero_rows(T* rows, int placed, const Rows& r) {
    constexpr int P = kPiece<T>;
    const int total = r.total;
    for (long long s = static_cast<long long>(min(max(placed, 0), total)) + blockIdx.x; s < total;
         s += gridDim.x) {
        T* row = rows + s * r.features;
        for (int c = threadIdx.x * P; c < r.features; c += 256 * P) {
            if (r.features - c >= P) store_piece(row + c, uint4{});
            else store_part(row + c, uint4{}, r.features - c);
        }
    }
}

// Copies rows of `features` T; WAVES waves of a workgroup share a token's row
// (WAVES = 1: the workgroup's four waves take a token each).  STREAM: past the caches.
template <typename T, int WAVES, bool STREAM>
__global__ __launch_bounds__(256) void tokens_dispatch(const T* __restrict__ x,
                                                       const int* __restrict__ slots,
                                                       const int* __restrict__ placed, Rows r,
                                                       T* __restrict__ xs) {
    constexpr int P = kPiece<T>, U = 4;
    const int wave  = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane  = (WAVES == 1 ? threadIdx.x & 63 : threadIdx.x) * P;
    const int step  = WAVES * 64 * P;
    const int total = r.total;
    const int t = blockIdx.x * (4 / WAVES) + (WAVES == 1 ? wave : 0);
    if (t < r.tokens) {
        const T* src = x + static_cast<long long>(t) * r.features;
        const int whole = r.features / P * P;
        for (int c = lane; c < whole; c += U * step) {
            uint4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (c + u * step < whole) v[u] = load_piece(src + c + u * step);
            }
            for (int j = 0; j < r.k; ++j) {
                const int s = slot_of(slots, static_cast<long long>(t) * r.k + j);
                if (static_cast<unsigned>(s) >= static_cast<unsigned>(total)) continue;
                T* dst = xs + static_cast<long long>(s) * r.features;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (c + u * step < whole) {
                        if constexpr (STREAM) stream_piece(dst + c + u * step, v[u]);
                        else store_piece(dst + c + u * step, v[u]);
                    }
                }
            }
        }
        if (lane == 0 && whole < r.features) {
            const uint4 v = load_part(src + whole, r.features - whole);
            for (int j = 0; j < r.k; ++j) {
                const int s = slots[static_cast<long long>(t) * r.k + j];
                if (static_cast<unsigned>(s) >= static_cast<unsigned>(total)) continue;
                store_part(xs + static_cast<long long>(s) * r.features + whole, v,
                           r.features - whole);
            }
        }
    }
    if (r.clear) zero_rows(xs, *placed, r);
}

// Sum over a token's slots, weighted where weights are given.  B slots' pieces
// are in flight at a time; an absent slot reads row 0 (which exists) and its
// value is dropped, so that nothing it holds, NaN included, reaches the sum.
template <typename T, int WAVES>
__global__ __launch_bounds__(256) void tokens_gather(const T* __restrict__ ys,
                                                     const int* __restrict__ slots,
                                                     const float* __restrict__ weights, Rows r,
                                                     T* __restrict__ y) {
    constexpr int P = kPiece<T>, B = 4;
    const int wave  = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane  = (WAVES == 1 ? threadIdx.x & 63 : threadIdx.x) * P;
    const int total = r.total;
    const int t = blockIdx.x * (4 / WAVES) + (WAVES == 1 ? wave : 0);
    if (t >= r.tokens) return;
    const long long e0 = static_cast<long long>(t) * r.k;
    for (int c = lane; c < r.features; c += WAVES * 64 * P) {
        float sum[P];
#pragma unroll
        for (int i = 0; i < P; ++i) sum[i] = 0.0f;
        const int count = min(P, r.features - c);
        for (int j0 = 0; j0 < r.k; j0 += B) {
            uint4 v[B];
            float w[B];
            bool  there[B];
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const int j = min(j0 + b, r.k - 1);
                const int s = slot_of(slots, e0 + j);
                there[b] = j0 + b < r.k && static_cast<unsigned>(s) < static_cast<unsigned>(total);
                w[b] = weights != nullptr ? weights[e0 + j] : 1.0f;
                const T* row = ys + static_cast<long long>(there[b] ? s : 0) * r.features + c;
                v[b] = count == P ? load_piece(row) : load_part(row, count);
            }
#pragma unroll
            for (int b = 0; b < B; ++b) {
                float f[P];
                piece_to_float<T>(v[b], f);
#pragma unroll
                for (int i = 0; i < P; ++i) sum[i] = there[b] ? fmaf(w[b], f[i], sum[i]) : sum[i];
            }
        }
        T* dst = y + static_cast<long long>(t) * r.features + c;
        const uint4 v = piece_from_float<T>(sum);
        if (count == P) store_piece(dst, v);
        else store_part(dst, v, count);
    }
}

template <typename T, int WAVES>
__global__ __launch_bounds__(256) void tokens_combine_grad(
    const T* __restrict__ dy, const T* __restrict__ ys, const int* __restrict__ slots,
    const int* __restrict__ placed, const float* __restrict__ weights, Rows r,
    T* __restrict__ dys, float* __restrict__ dweights) {
    constexpr int P = kPiece<T>, B = 4;
    __shared__ float s_part[4][B];
    const int wave  = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane  = (WAVES == 1 ? threadIdx.x & 63 : threadIdx.x) * P;
    const int total = r.total;
    const int t = blockIdx.x * (4 / WAVES) + (WAVES == 1 ? wave : 0);
    const long long e0 = static_cast<long long>(t) * r.k;
    const T* src = dy + static_cast<long long>(t) * r.features;
    // with WAVES = 4 all waves have the same token: the barriers below are met by all
    for (int j0 = 0; t < r.tokens && j0 < r.k; j0 += B) {
        int   s[B];
        float w[B], dot[B];
        bool  there[B];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const int j = min(j0 + b, r.k - 1);
            s[b] = slot_of(slots, e0 + j);
            there[b] = j0 + b < r.k && static_cast<unsigned>(s[b]) < static_cast<unsigned>(total);
            s[b] = there[b] ? s[b] : 0;
            w[b] = weights[e0 + j];
            dot[b] = 0.0f;
        }
        for (int c = lane; c < r.features; c += WAVES * 64 * P) {
            const int count = min(P, r.features - c);
            uint4 v[B];
            const uint4 g = count == P ? load_piece(src + c) : load_part(src + c, count);
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const T* row = ys + static_cast<long long>(s[b]) * r.features + c;
                v[b] = count == P ? load_piece(row) : load_part(row, count);
            }
            float gf[P];
            piece_to_float<T>(g, gf);
#pragma unroll
            for (int b = 0; b < B; ++b) {
                float f[P];
                piece_to_float<T>(v[b], f);
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    dot[b] = fmaf(gf[i], f[i], dot[b]);
                    f[i] = w[b] * gf[i];
                }
                if (there[b]) {
                    T* dst = dys + static_cast<long long>(s[b]) * r.features + c;
                    const uint4 o = piece_from_float<T>(f);
                    if (count == P) store_piece(dst, o);
                    else store_part(dst, o, count);
                }
            }
        }
#pragma unroll
        for (int b = 0; b < B; ++b) dot[b] = wave_sum(dot[b]);
        if constexpr (WAVES == 4) {
            if ((threadIdx.x & 63) == 0) {
#pragma unroll
                for (int b = 0; b < B; ++b) s_part[wave][b] = dot[b];
            }
            __syncthreads();
#pragma unroll
            for (int b = 0; b < B; ++b) {
                dot[b] = (s_part[0][b] + s_part[1][b]) + (s_part[2][b] + s_part[3][b]);
            }
            __syncthreads();
        }
        if (lane == 0) {
#pragma unroll
            for (int b = 0; b < B; ++b) {
                if (j0 + b < r.k) dweights[e0 + j0 + b] = there[b] ? dot[b] : 0.0f;
            }
        }
    }
    if (r.clear) zero_rows(dys, *placed, r);
}

Error check_rows(int tokens, int k, int features, const char* name) {
    if (tokens < 0 || k < 1 || features < 0) {
        return Error{kInvalid, std::string(name) + ": sizes must be positive"};
    }
    if (static_cast<long long>(tokens) * k > 0x3fffffffLL) {
        return Error{kUnsupported, std::string(name) + ": over 2^30 entries"};
    }
    // a step past a row's last column has to stay an int
    if (features > 0x7fff0000) {
        return Error{kUnsupported, std::string(name) + ": rows over 2^31 - 2^16 elements"};
    }
    return Error{};
}

// One wave a token fills the chip's 1024 SIMDs from about this many tokens on; below, four
// waves share a token.  Measured both ways over 126 sizes: 8192 tokens x 8 x 128 bf16 5.9,
// 7.2 and 11.6 us (dispatch, combine, combine_backward) with one wave, 7.5, 9.0 and 25.1
// with four; 1024 x 1 x 7168 4.9, 14.5 and 14.2, 4.7, 8.6 and 8.1.  Rows of 8 KB and more
// are up to 15% faster with four waves past it too.
constexpr int kWaveTokens = 4096;

// Rows that the 256 MB cache in front of memory cannot hold are stored past it: 8192
// tokens x 8 x 4096 bf16 (512 MB) take 106 us, 120 with plain stores; 5003 x 4 x 2050
// (80 MB), which the cache holds for the next reader, 17 us with plain stores, 22 so.
constexpr long long kStreamBytes = 256LL << 20;

// Calls f(element, waves a token, first token, rows, workgroups) for each launch: 67 M
// tokens of a wave each are as many as one has threads for.
template <typename F>
Error with_shape(ElementType type, int tokens, int k, int features, F f) {
    auto waves = [&](auto zero) {
        const int total = tokens * k;
        if (tokens < kWaveTokens) {
            return f(zero, std::integral_constant<int, 4>{}, 0LL, Rows{tokens, k, features, total, true},
                     tokens);
        }
        constexpr long long most = kLaunchThreads / 256 * 4;
        for (long long first = 0; first < tokens; first += most) {
            const int here = static_cast<int>(std::min(most, tokens - first));
            SPMM_TRY(f(zero, std::integral_constant<int, 1>{}, first,
                       Rows{here, k, features, total, first == 0}, (here + 3) / 4));
        }
        return Error{};
    };
    switch (type) {
        case ElementType::F32: return waves(float{});
        case ElementType::F16: return waves(_Float16{});
        case ElementType::BF16: return waves(__bf16{});
    }
    return Error{kInvalid, "unknown element type"};
}

}  // namespace

Error launch_dispatch(const void* x, ElementType type, int tokens, int k, int features,
                      const int* slots, const int* offsets, int experts, void* xs,
                      hipStream_t stream) {
    SPMM_TRY(check_rows(tokens, k, features, "dispatch"));
    if (experts < 1) return Error{kInvalid, "dispatch: sizes must be positive"};
    if (tokens == 0 || features == 0) return Error{};
    if (x == nullptr || slots == nullptr || offsets == nullptr || xs == nullptr) {
        return Error{kInvalid, "dispatch: null pointer"};
    }
    return with_shape(type, tokens, k, features, [&](auto zero, auto waves, long long first, Rows r,
                                                     int blocks) {
        using T = decltype(zero);
        const bool past = static_cast<long long>(tokens) * k * features * sizeof(T) >= kStreamBytes;
        auto kernel = past ? tokens_dispatch<T, waves.value, true>
                           : tokens_dispatch<T, waves.value, false>;
        kernel<<<blocks, 256, 0, stream>>>(static_cast<const T*>(x) + first * features,
                                           slots + first * k, offsets + experts, r,
                                           static_cast<T*>(xs));
        SPMM_TRY_HIP(hipGetLastError(), "dispatch");
        return Error{};
    });
}

Error launch_combine(const void* ys, ElementType type, int tokens, int k, int features,
                     const int* slots, const float* weights, void* y, hipStream_t stream) {
    SPMM_TRY(check_rows(tokens, k, features, "combine"));
    if (tokens == 0 || features == 0) return Error{};
    if (ys == nullptr || slots == nullptr || y == nullptr) {
        return Error{kInvalid, "combine: null pointer"};
    }
    return with_shape(type, tokens, k, features, [&](auto zero, auto waves, long long first, Rows r,
                                                     int blocks) {
        using T = decltype(zero);
        tokens_gather<T, waves.value><<<blocks, 256, 0, stream>>>(
            static_cast<const T*>(ys), slots + first * k,
            weights != nullptr ? weights + first * k : nullptr, r,
            static_cast<T*>(y) + first * features);
        SPMM_TRY_HIP(hipGetLastError(), "combine");
        return Error{};
    });
}

Error launch_combine_backward(const void* dy, const void* ys, ElementType type, int tokens, int k,
                              int features, const int* slots, const float* weights,
                              const int* offsets, int experts, void* dys, float* dweights,
                              hipStream_t stream) {
    SPMM_TRY(check_rows(tokens, k, features, "combine_backward"));
    if (experts < 1) return Error{kInvalid, "combine_backward: sizes must be positive"};
    if (tokens == 0) return Error{};
    if (slots == nullptr || weights == nullptr || offsets == nullptr || dweights == nullptr ||
        (features > 0 && (dy == nullptr || ys == nullptr || dys == nullptr))) {
        return Error{kInvalid, "combine_backward: null pointer"};
    }
    return with_shape(type, tokens, k, features, [&](auto zero, auto waves, long long first, Rows r,
                                                     int blocks) {
        using T = decltype(zero);
        tokens_combine_grad<T, waves.value><<<blocks, 256, 0, stream>>>(
            static_cast<const T*>(dy) + first * features, static_cast<const T*>(ys),
            slots + first * k, offsets + experts, weights + first * k, r, static_cast<T*>(dys),
            dweights + first * k);
        SPMM_TRY_HIP(hipGetLastError(), "combine_backward");
        return Error{};
    });
}

}  // namespace engine
}  // namespace spmm
