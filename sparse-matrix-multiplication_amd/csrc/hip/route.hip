// Routing of tokens to experts: the k largest logits of each token with their
// softmax weights, and the order of the (token, choice) entries by expert -- the
// routing matrix's rows (k entries a token) and its transpose's order.
//
//   C_t = the k largest of logits[t] (ties: the lowest expert; -inf is never chosen)
//   w_j = exp(l_j - m) / sum exp(l_i - m), over C_t or over all experts, m the largest
//   gradient: over C_t  dl_j = w_j (dw_j - D), over all  dl_e = p_e ([e in C] dw_e - D),
//             D = sum_j w_j dw_j
//
// The order is a counting sort in two launches: blocks count their entries by
// expert while they choose (or from given ids), then every block places its own
// entries from all blocks' counts.  Places follow from counts alone, never from
// the order of atomics, so equal experts keep their entries' order.
//
// Few tokens are one block's, which chooses and places in one launch: a call for one
// token of 64 experts, k = 6, is then bound by its host side (15.8 us; 18.5 with two
// launches).

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

constexpr int kMaxGroups   = 1024;  // a place block's running starts fit the LDS
constexpr int kMaxChoices  = 64;    // one lane holds one choice
constexpr int kChooseWaves = 16;
constexpr int kPlaceWaves  = 8;

// A float as an unsigned whose order is the floats' order: NaN above all, -0
// equal to +0, nothing at or below kNone is ever chosen (-inf, or no element).
constexpr unsigned kNone = 0x007fffffu;
__device__ __forceinline__ unsigned key_of(float f) {
    unsigned u = __float_as_uint(f);
    u = f != f ? 0x7fffffffu : f == 0.0f ? 0u : u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(unsigned k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// For 16-bit logits a key holds both: the value's order in the upper half and the
// expert, counted down, in the lower, so that one maximum finds the largest value
// at its lowest expert.  Four tokens share a wave, sixteen lanes each.
__device__ __forceinline__ unsigned order16(unsigned bits, bool nan) {
    bits = nan ? 0x7fffu : (bits & 0x7fffu) == 0 ? 0u : bits;
    return bits & 0x8000u ? ~bits & 0xffffu : bits | 0x8000u;
}
__device__ __forceinline__ unsigned row_max(unsigned v) {
    // rotations of each row of sixteen lanes: every lane ends with the row's largest
#define SPMM_STEP(C) { const unsigned o = dpp<C>(0u, v); v = v > o ? v : o; }
    SPMM_STEP(0x128) SPMM_STEP(0x124) SPMM_STEP(0x122) SPMM_STEP(0x121)
#undef SPMM_STEP
    return v;
}
__device__ __forceinline__ float row_sum(float v) {
#define SPMM_STEP(C) v += __uint_as_float(dpp<C>(0u, __float_as_uint(v)));
    SPMM_STEP(0x128) SPMM_STEP(0x124) SPMM_STEP(0x122) SPMM_STEP(0x121)
#undef SPMM_STEP
    return v;
}

template <typename T, int PER>
__device__ __forceinline__ void load_logits(const T* row, int experts, float (&v)[PER]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = i * 64 + lane;
        v[i] = e < experts ? static_cast<float>(row[e]) : -__builtin_inff();
    }
}

// One wave chooses for one token: lane j < k leaves with choice j and its weight.  16384
// tokens, 128 experts, k = 8, fp32: 12.9 us, bound by the k maxima, a chain over 64 lanes
// each.
template <int PER>
__device__ __forceinline__ void choose(const float (&v)[PER], int k, bool all, int& expert,
                                       float& weight) {
    const int lane = threadIdx.x & 63;
    unsigned key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = key_of(v[i]);
    expert = -1;
    float value = -__builtin_inff(), largest = 0.0f;
    for (int j = 0; j < k; ++j) {
        unsigned m = key[0];
#pragma unroll
        for (int i = 1; i < PER; ++i) m = m > key[i] ? m : key[i];
        m = wave_max(m);
        if (m <= kNone) break;
        // experts i * 64 + lane: the lowest is in the first register that holds m
        int e = -1;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const unsigned long long at = __ballot(key[i] == m);
            if (e < 0 && at != 0) {
                e = i * 64 + __builtin_ctzll(at);
                if (lane == (e & 63)) key[i] = 0u;
            }
        }
        const float f = key_value(m);
        if (j == 0) largest = f;
        if (lane == j) {
            expert = e;
            value  = f;
        }
    }
    const float mine = expert >= 0 ? expf(value - largest) : 0.0f;
    float part = mine;
    if (all) {
        part = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) part += expf(v[i] - largest);
    }
    const float total = wave_sum(part);
    weight = expert >= 0 ? mine / total : 0.0f;
}

// Counts of one block: chunk b of the entries, by expert.
struct Order {
    const int* ids;      // n expert ids; those outside [0, groups) have no place
    int        n;
    int        groups;
    int        chunk;    // entries a block
    int*       counts;   // blocks x groups
    int*       offsets;  // groups + 1
    int*       entries;  // n
    int*       slots;    // n
};

// Places chunk b: entry i of expert e goes to offsets[e] + (entries of e in
// earlier chunks) + (in earlier waves' parts) + (in earlier rounds and lanes).
// Every block sums the other blocks' counts itself: blocks x groups ints from
// L2 a block, less than a third launch between the two would cost (131072 entries of
// 128 experts: 6.8 us, most of it this chain of waits and 256 x 128 counts a block).
// A block that is alone counts its own entries and reads nobody's.
template <int WAVES>
__device__ __forceinline__ void place_chunk(const Order& o, int* s) {
    int* s_start = s;                     // kPlaceWaves x groups: next place, by wave
    int* s_total = s + kPlaceWaves * o.groups;
    int* s_before = s_total + o.groups;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr int threads = WAVES * 64;  // those past kPlaceWaves have no entries
    for (int i = threadIdx.x; i < (kPlaceWaves + 2) * o.groups; i += threads) s[i] = 0;
    __syncthreads();

    // counts of all blocks and of the earlier ones: `parts` threads share a column
    const int parts = max(1, threads / o.groups);
    const int blocks = gridDim.x;
    for (int i = threadIdx.x; blocks > 1 && i < parts * o.groups; i += threads) {
        const int g = i % o.groups;
        int total = 0, before = 0;
#pragma unroll 16
        for (int b = i / o.groups; b < blocks; b += parts) {
            const int c = o.counts[static_cast<long long>(b) * o.groups + g];
            total += c;
            before += b < static_cast<int>(blockIdx.x) ? c : 0;
        }
        atomicAdd(&s_total[g], total);
        atomicAdd(&s_before[g], before);
    }
    // this block's own entries by wave
    const int part = (o.chunk + kPlaceWaves - 1) / kPlaceWaves;
    const int c1 = min((static_cast<int>(blockIdx.x) + 1) * o.chunk, o.n);
    const int i0 = min(static_cast<int>(blockIdx.x) * o.chunk + wave * part, c1);
    const int i1 = min(i0 + part, c1);
    for (int i = i0 + lane; i < i1; i += 64) {
        const int id = o.ids[i];
        if (static_cast<unsigned>(id) < static_cast<unsigned>(o.groups)) {
            atomicAdd(&s_start[wave * o.groups + id], 1);
        }
    }
    __syncthreads();
    if (blocks == 1) {
        for (int g = threadIdx.x; g < o.groups; g += threads) {
            int c = 0;
            for (int w = 0; w < kPlaceWaves; ++w) c += s_start[w * o.groups + g];
            s_total[g] = c;
        }
        __syncthreads();
    }
    // s_total becomes each group's first place
    if (wave == 0) {
        int run = 0;
        for (int g0 = 0; g0 < o.groups; g0 += 64) {
            const int g = g0 + lane;
            const int c = g < o.groups ? s_total[g] : 0;
            const int upto = wave_prefix(c);
            if (g < o.groups) s_total[g] = run + upto - c;
            run += __shfl(upto, 63);
        }
        if (lane == 0) s[(kPlaceWaves + 2) * o.groups] = run;
    }
    __syncthreads();
    const int placed = s[(kPlaceWaves + 2) * o.groups];
    if (blockIdx.x == 0) {
        for (int g = threadIdx.x; g < o.groups; g += threads) o.offsets[g] = s_total[g];
        if (threadIdx.x == 0) o.offsets[o.groups] = placed;
    }
    for (int g = threadIdx.x; g < o.groups; g += threads) {
        int at = s_total[g] + s_before[g];
        for (int w = 0; w < kPlaceWaves; ++w) {
            const int c = s_start[w * o.groups + g];
            s_start[w * o.groups + g] = at;
            at += c;
        }
    }
    __syncthreads();

    volatile int* start = s_start + wave * o.groups;
    for (int at = i0; at < i1; at += 64) {
        const int i = at + lane;
        const int id = i < i1 ? o.ids[i] : -1;
        const bool in = static_cast<unsigned>(id) < static_cast<unsigned>(o.groups);
        // lanes of this round with the same id, one ballot a bit of the id
        unsigned long long same = __ballot(in);
        for (int b = 1; b < o.groups; b *= 2) {
            const unsigned long long set = __ballot((id & b) != 0);
            same &= (id & b) != 0 ? set : ~set;
        }
        if (in) {
            const int rank = __builtin_popcountll(same & ((1ull << lane) - 1));
            const int slot = start[id] + rank;
            __builtin_amdgcn_wave_barrier();  // all lanes have read before the last one counts up
            if (same >> lane == 1) start[id] = slot + 1;
            o.slots[i] = slot;
            o.entries[slot] = i;
        } else if (i < i1) {
            o.slots[i] = -1;
        }
        __builtin_amdgcn_wave_barrier();
    }
    for (int i = placed + blockIdx.x * threads + threadIdx.x; i < o.n; i += gridDim.x * threads) {
        o.entries[i] = -1;
    }
}

template <typename T, int PER, bool ALONE>
__global__ __launch_bounds__(kChooseWaves * 64) void route_choose(
    const T* __restrict__ logits, int tokens, int experts, int k, int all, int per_block,
    float* __restrict__ out_weights, int* out_experts, Order order) {
    extern __shared__ int s_count[];
    if constexpr (!ALONE) {
        for (int e = threadIdx.x; e < experts; e += blockDim.x) s_count[e] = 0;
        __syncthreads();
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t1 = min((static_cast<int>(blockIdx.x) + 1) * per_block, tokens);
    for (int t = blockIdx.x * per_block + wave; t < t1; t += kChooseWaves) {
        float v[PER];
        load_logits<T, PER>(logits + static_cast<long long>(t) * experts, experts, v);
        int   expert;
        float weight;
        choose<PER>(v, k, all != 0, expert, weight);
        if (lane < k) {
            out_experts[static_cast<long long>(t) * k + lane] = expert;
            out_weights[static_cast<long long>(t) * k + lane] = weight;
            if (!ALONE && expert >= 0) atomicAdd(&s_count[expert], 1);
        }
    }
    __syncthreads();
    if constexpr (ALONE) {
        place_chunk<kChooseWaves>(order, s_count);
    } else {
        for (int e = threadIdx.x; e < experts; e += blockDim.x) {
            order.counts[static_cast<long long>(blockIdx.x) * experts + e] = s_count[e];
        }
    }
}

// route_choose for 16-bit logits and k <= 16: the token's lane j < k holds choice j.
// 16384 tokens, 128 experts, k = 8: 6.7 us, one token a wave 14.5.
template <typename T, int PER, bool ALONE>
__global__ __launch_bounds__(kChooseWaves * 64) void route_choose_quads(
    const T* __restrict__ logits, int tokens, int experts, int k, int all, int per_block,
    float* __restrict__ out_weights, int* out_experts, Order order) {
    extern __shared__ int s_count[];
    if constexpr (!ALONE) {
        for (int e = threadIdx.x; e < experts; e += blockDim.x) s_count[e] = 0;
        __syncthreads();
    }
    const int lane = threadIdx.x & 15;
    const int t1 = min((static_cast<int>(blockIdx.x) + 1) * per_block, tokens);
    // whole waves stay together: the rotations need all lanes of a row
    for (int t0 = blockIdx.x * per_block; t0 < t1; t0 += kChooseWaves * 4) {
        const int t = t0 + static_cast<int>(threadIdx.x >> 4);
        unsigned key[PER];
        float v[PER];
        const T* row = logits + static_cast<long long>(t < t1 ? t : t1 - 1) * experts;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = i * 16 + lane;
            const T x = e < experts ? row[e] : static_cast<T>(0.0f);
            v[i] = e < experts ? static_cast<float>(x) : -__builtin_inff();
            const bool none = v[i] == -__builtin_inff();
            key[i] = none ? 0u : order16(__builtin_bit_cast(unsigned short, x), v[i] != v[i]) << 16 |
                                     (0xffffu - e);
        }
        int expert = -1;
        unsigned mine = 0u, first = 0u;
        for (int j = 0; j < k; ++j) {
            unsigned m = key[0];
#pragma unroll
            for (int i = 1; i < PER; ++i) m = m > key[i] ? m : key[i];
            m = row_max(m);
#pragma unroll
            for (int i = 0; i < PER; ++i) key[i] = key[i] == m ? 0u : key[i];
            first = j == 0 ? m : first;
            mine = lane == j ? m : mine;
        }
        auto value = [](unsigned m) {
            const unsigned u = m >> 16;
            const unsigned short bits = static_cast<unsigned short>(u & 0x8000u ? u & 0x7fffu : ~u);
            return static_cast<float>(__builtin_bit_cast(T, bits));
        };
        const float largest = first != 0u ? value(first) : 0.0f;
        expert = mine != 0u ? static_cast<int>(0xffffu - (mine & 0xffffu)) : -1;
        const float e = mine != 0u ? expf(value(mine) - largest) : 0.0f;
        float part = e;
        if (all) {
            part = 0.0f;
#pragma unroll
            for (int i = 0; i < PER; ++i) part += expf(v[i] - largest);
        }
        const float total = row_sum(part);
        if (lane < k && t < t1) {
            out_experts[static_cast<long long>(t) * k + lane] = expert;
            out_weights[static_cast<long long>(t) * k + lane] = expert >= 0 ? e / total : 0.0f;
            if (!ALONE && expert >= 0) atomicAdd(&s_count[expert], 1);
        }
    }
    __syncthreads();
    if constexpr (ALONE) {
        place_chunk<kChooseWaves>(order, s_count);
    } else {
        for (int e = threadIdx.x; e < experts; e += blockDim.x) {
            order.counts[static_cast<long long>(blockIdx.x) * experts + e] = s_count[e];
        }
    }
}

__global__ __launch_bounds__(256) void group_count(Order o) {
    extern __shared__ int s_count[];
    for (int g = threadIdx.x; g < o.groups; g += 256) s_count[g] = 0;
    __syncthreads();
    const int i1 = min((static_cast<int>(blockIdx.x) + 1) * o.chunk, o.n);
    for (int i = blockIdx.x * o.chunk + threadIdx.x; i < i1; i += 256) {
        const int id = o.ids[i];
        if (static_cast<unsigned>(id) < static_cast<unsigned>(o.groups)) atomicAdd(&s_count[id], 1);
    }
    __syncthreads();
    for (int g = threadIdx.x; g < o.groups; g += 256) {
        o.counts[static_cast<long long>(blockIdx.x) * o.groups + g] = s_count[g];
    }
}

__global__ __launch_bounds__(kPlaceWaves * 64) void group_place(Order o) {
    extern __shared__ int s[];
    place_chunk<kPlaceWaves>(o, s);
}

// A wave a token: the softmax again from the logits where it runs over all experts.
// 8191 tokens of 100 experts, fp32: 5.2 us, 1.3 TB/s.  Bound by its form: a token's three
// reductions over 64 lanes are chains of six dependent steps, and a wave has one token
// (sixteen lanes a token, as route_choose_quads has them, are not built for it).
template <typename T, int PER>
__global__ __launch_bounds__(256) void route_grad(const T* __restrict__ logits, int tokens,
                                                  int experts, int k, int all,
                                                  const int* __restrict__ chosen,
                                                  const float* __restrict__ weights,
                                                  const float* __restrict__ dweights,
                                                  T* __restrict__ dlogits) {
    const int lane = threadIdx.x & 63;
    const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= tokens) return;
    const long long at = static_cast<long long>(t) * k + lane;
    const int   e  = lane < k ? chosen[at] : -1;
    const float w  = e >= 0 ? weights[at] : 0.0f;
    const float dw = e >= 0 ? dweights[at] : 0.0f;
    const float dot = wave_sum(w * dw);
    float d[PER];
    const long long row = static_cast<long long>(t) * experts;
    if (all) {
        float v[PER];
        load_logits<T, PER>(logits + row, experts, v);
        unsigned m = 0u;
#pragma unroll
        for (int i = 0; i < PER; ++i) m = max(m, key_of(v[i]));
        m = wave_max(m);
        const float largest = m > kNone ? key_value(m) : 0.0f;
        float part = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            v[i] = expf(v[i] - largest);
            part += v[i];
            d[i] = -dot;
        }
        const float total = wave_sum(part);
        for (int j = 0; j < k; ++j) {
            const int   ej = __builtin_amdgcn_readlane(e, j);
            const float dj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(dw), j));
#pragma unroll
            for (int i = 0; i < PER; ++i) d[i] += i * 64 + lane == ej ? dj : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) d[i] *= total == 0.0f ? 0.0f : v[i] / total;
    } else {
        const float mine = w * (dw - dot);
#pragma unroll
        for (int i = 0; i < PER; ++i) d[i] = 0.0f;
        for (int j = 0; j < k; ++j) {
            const int   ej = __builtin_amdgcn_readlane(e, j);
            const float dj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mine), j));
#pragma unroll
            for (int i = 0; i < PER; ++i) d[i] += i * 64 + lane == ej ? dj : 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (i * 64 + lane < experts) dlogits[row + i * 64 + lane] = static_cast<T>(d[i]);
    }
}

// Entries a block of the sort: at most 256 blocks, whose counts every block
// reads, and at least 512 entries, so that placing outweighs reading them.
int chunk_of(long long n) {
    const long long c = (n + 255) / 256;
    return static_cast<int>(std::max<long long>(512, (c + 63) / 64 * 64));
}
int blocks_of(long long n, int chunk) {
    return static_cast<int>((n + chunk - 1) / chunk);
}

Error check_sizes(int tokens, int experts, int k) {
    if (tokens < 0 || experts < 1 || k < 1) return Error{kInvalid, "route: sizes must be positive"};
    if (k > experts) return Error{kInvalid, "route: k exceeds the number of experts"};
    if (experts > kMaxGroups) return Error{kUnsupported, "route: at most 1024 experts"};
    if (k > kMaxChoices) return Error{kUnsupported, "route: at most 64 experts a token"};
    if (static_cast<long long>(tokens) * k > 0x3fffffffLL) {
        return Error{kUnsupported, "route: over 2^30 entries"};
    }
    return Error{};
}

size_t place_lds(int groups) { return sizeof(int) * ((kPlaceWaves + 2) * groups + 1); }
Error place(Order o, int blocks, hipStream_t stream) {
    group_place<<<blocks, kPlaceWaves * 64, place_lds(o.groups), stream>>>(o);
    SPMM_TRY_HIP(hipGetLastError(), "group_place");
    return Error{};
}

// No entries: every offset is 0.
__global__ void zero_ints(int* p, int n) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) p[i] = 0;
}
Error no_entries(int groups, int* offsets, hipStream_t stream) {
    zero_ints<<<1, 256, 0, stream>>>(offsets, groups + 1);
    SPMM_TRY_HIP(hipGetLastError(), "group_place");
    return Error{};
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

// Elements a lane holds of `experts` logits.
template <typename F>
void with_per(int experts, F f) {
    if (experts <= 64) f(std::integral_constant<int, 1>{});
    else if (experts <= 128) f(std::integral_constant<int, 2>{});
    else if (experts <= 256) f(std::integral_constant<int, 4>{});
    else if (experts <= 512) f(std::integral_constant<int, 8>{});
    else f(std::integral_constant<int, 16>{});
}

// 16-bit logits of few experts and choices go four tokens a wave.
bool four_a_wave(ElementType type, int experts, int k) {
    return type != ElementType::F32 && k <= 16 && experts <= 256;
}

// Tokens a block that chooses takes: at most about a chunk of the sort's entries, and so
// few rounds of its waves (two, or one of four tokens a wave) that a block a CU shares them
// before a block takes more.  16384 tokens of 64 experts, fp32, k = 1: 9.6 us, 28.4 with
// chunks of entries alone; 512 tokens 7.3, 24.5 in one block; of 1024 experts 17.1, 83.
// What one block does in less time than a second launch takes is left to it: 64 tokens of 64
// experts, fp32, k = 1 5.7 us, 7.0 in two blocks; of 1024 experts, k = 8 43, 29 so.
int tokens_per_block(long long tokens, int experts, int k, bool four) {
    long long t = (chunk_of(tokens * k) + k - 1) / k;
    if (tokens > (four ? 128 : k <= 4 && experts <= 256 ? 64 : 48)) {
        t = std::min(t, std::max<long long>(four ? 64 : 32, (tokens + 255) / 256));
    }
    return static_cast<int>((t + kChooseWaves - 1) / kChooseWaves * kChooseWaves);
}

}  // namespace

long long group_workspace(long long entries, int groups) {
    if (entries <= 0 || groups < 1) return 0;
    return static_cast<long long>(sizeof(int)) * groups * blocks_of(entries, chunk_of(entries));
}

long long route_workspace(long long tokens, int experts, int k) {
    if (tokens <= 0 || experts < 1 || k < 1) return 0;
    // the counts of any element type: one token a wave has the more blocks
    return static_cast<long long>(sizeof(int)) * experts *
           blocks_of(tokens, tokens_per_block(tokens, experts, k, false));
}

Error launch_group_entries(const int* ids, int n, int groups, int* offsets, int* entries,
                           int* slots, void* workspace, hipStream_t stream) {
    if (n < 0 || groups < 1) return Error{kInvalid, "group_entries: sizes must be positive"};
    if (groups > kMaxGroups) return Error{kUnsupported, "group_entries: at most 1024 groups"};
    if (n > 0x3fffffff) return Error{kUnsupported, "group_entries: over 2^30 entries"};
    if (offsets == nullptr) return Error{kInvalid, "group_entries: null offsets"};
    if (n == 0) return no_entries(groups, offsets, stream);
    const Order o{ids, n, groups, chunk_of(n), static_cast<int*>(workspace), offsets, entries, slots};
    const int blocks = blocks_of(n, o.chunk);
    if (ids == nullptr || entries == nullptr || slots == nullptr || workspace == nullptr) {
        return Error{kInvalid, "group_entries: null pointer"};
    }
    if (blocks == 1) return place(o, 1, stream);
    group_count<<<blocks, 256, sizeof(int) * groups, stream>>>(o);
    SPMM_TRY_HIP(hipGetLastError(), "group_count");
    return place(o, blocks, stream);
}

Error launch_route(const void* logits, ElementType type, int tokens, int experts, int k, bool all,
                   int* out_experts, float* out_weights, int* offsets, int* entries, int* slots,
                   void* workspace, hipStream_t stream) {
    SPMM_TRY(check_sizes(tokens, experts, k));
    if (offsets == nullptr) return Error{kInvalid, "route: null offsets"};
    if (tokens == 0) return no_entries(experts, offsets, stream);
    const bool four = four_a_wave(type, experts, k);
    const int per = tokens_per_block(tokens, experts, k, four);
    const int blocks = blocks_of(tokens, per);
    if (logits == nullptr || out_experts == nullptr || out_weights == nullptr ||
        entries == nullptr || slots == nullptr || workspace == nullptr) {
        return Error{kInvalid, "route: null pointer"};
    }
    const Order order{out_experts, tokens * k, experts, per * k, static_cast<int*>(workspace),
                      offsets, entries, slots};
    const bool alone = blocks == 1;
    SPMM_TRY(with_type(type, [&](auto zero) {
        using T = decltype(zero);
        auto launch = [&](auto kernel) {
            kernel<<<blocks, kChooseWaves * 64, alone ? place_lds(experts) : sizeof(int) * experts,
                     stream>>>(static_cast<const T*>(logits), tokens, experts, k, all ? 1 : 0, per,
                               out_weights, out_experts, order);
        };
        if constexpr (sizeof(T) == 2) {
            if (four) {
                auto quads = [&](auto n) {
                    launch(alone ? route_choose_quads<T, n.value, true>
                                 : route_choose_quads<T, n.value, false>);
                };
                if (experts <= 64) quads(std::integral_constant<int, 4>{});
                else if (experts <= 128) quads(std::integral_constant<int, 8>{});
                else quads(std::integral_constant<int, 16>{});
                SPMM_TRY_HIP(hipGetLastError(), "route_choose");
                return Error{};
            }
        }
        with_per(experts, [&](auto n) {
            launch(alone ? route_choose<T, n.value, true> : route_choose<T, n.value, false>);
        });
        SPMM_TRY_HIP(hipGetLastError(), "route_choose");
        return Error{};
    }));
    return alone ? Error{} : place(order, blocks, stream);
}

Error launch_route_backward(const void* logits, ElementType type, int tokens, int experts, int k,
                            bool all, const int* chosen, const float* weights,
                            const float* dweights, void* dlogits, hipStream_t stream) {
    SPMM_TRY(check_sizes(tokens, experts, k));
    if (tokens == 0) return Error{};
    if ((all && logits == nullptr) || chosen == nullptr || weights == nullptr ||
        dweights == nullptr || dlogits == nullptr) {
        return Error{kInvalid, "route_backward: null pointer"};
    }
    return with_type(type, [&](auto zero) {
        using T = decltype(zero);
        // 67 M tokens of a wave each are as many as one launch has threads for
        constexpr long long most = kLaunchThreads / 256 * 4;
        for (long long first = 0; first < tokens; first += most) {
            const int here = static_cast<int>(std::min(most, tokens - first));
            with_per(experts, [&](auto n) {
                route_grad<T, n.value><<<(here + 3) / 4, 256, 0, stream>>>(
                    all ? static_cast<const T*>(logits) + first * experts : nullptr, here, experts, k,
                    all ? 1 : 0, chosen + first * k, weights + first * k, dweights + first * k,
                    static_cast<T*>(dlogits) + first * experts);
            });
            SPMM_TRY_HIP(hipGetLastError(), "route_grad");
        }
        return Error{};
    });
}

}  // namespace engine
}  // namespace spmm
