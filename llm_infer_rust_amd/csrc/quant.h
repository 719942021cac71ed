// Row quantisation shared by the 8-bit projections (quant.hip) and the 8-bit experts (experts.hip).
#pragma once

#include "product.h"

namespace mi355x {

// values[r, :] and scales[r] of `rows` rows of `width` elements (dtype 0 bf16, 1 fp16, 2 fp32), row
// stride in bytes. Columns up to the next multiple of 16 are written as zeros.
const char* run_quantize_rows(const void* x, int64_t stride, void* values, int64_t ldv,
                              float* scales, int64_t rows, int64_t width, int dtype,
                              hipStream_t s);

}  // namespace mi355x
