// Products in 8-bit integers, a scale a row of either operand:
//
//   out[s, c] = sx[s] sw[c] sum_k qx[s, k] qw[c, k]
//
// The tile kernels and the kernel for few rows with v_mfma_i32_16x16x64_i8: its operands
// are as many bytes a lane as those of the 16-bit products, so rows of integers are moved
// as rows of half as many pairs, and a step of the contraction does twice the work.  Sums
// are exact in 32 bits; they are scaled in fp32 on their way out and rounded once.

#include <hip/hip_runtime.h>

#include "tile_products.h"

namespace spmm {
namespace engine {

Error launch_int8_mm(const void* x, const float* x_scales, const void* w, const float* w_scales,
                     const int* offsets, int groups, int total, int width, int depth,
                     ElementType out_type, void* out, hipStream_t stream) {
    TileArgs a{};
    SPMM_TRY(int8_args(x, x_scales, w, w_scales, offsets, groups, total, width, depth, out_type, out,
                       "int8_mm", a));
    if (total == 0) return Error{};
    return launch_finished<Int8Pair, Ends::Plain>(a, Lie::Pieces, stream, "int8_mm");
}

}  // namespace engine
}  // namespace spmm
