// Launch functions of the block-scaled 8-bit kernels; nnf_api.hip checks what it is given before calling in.
#pragma once

#include "fp8.h"

namespace nnf
{
    // index == null: every row; else row i of the results is x's row index[i], zeros where there is no such row
    hipError_t launch_fp8_quantize(hipStream_t s, const void* x, bool bf16, const void* index, void* codes, float* scales, int rows, int source_rows, int K);
    hipError_t launch_fp8_quantize_weights(hipStream_t s, const void* w, bool bf16, void* codes, float* scales, int matrices, int N, int K);
    // `kernel`: one of fp8::Kernel, those up to TILE_256x256, then the others
    hipError_t launch_fp8_tiles(hipStream_t s, const fp8::Operands& o, int kernel, bool gate);
    hipError_t launch_fp8_rows(hipStream_t s, const fp8::Operands& o, int kernel, bool gate);
} // namespace nnf
