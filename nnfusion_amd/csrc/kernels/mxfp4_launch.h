// Launch functions of the MXFP4 kernels; nnf_api.hip checks what it is given before calling in.
#pragma once

#include "mxfp4.h"

namespace nnf
{
    // rows == null: every row; else codes and scales of row i are those of x's row index[i], zeros where there is no such row
    hipError_t launch_mxfp4_quantize(hipStream_t s, const void* x, const void* index, void* codes, void* scales, int rows, int source_rows, int K);
    hipError_t launch_mxfp4_dequantize(hipStream_t s, const void* codes, const void* scales, void* y, int rows, int K);
    // `kernel`: one of mx::Kernel that has this form (mx::choose)
    hipError_t launch_mxfp4_rows(hipStream_t s, const mx::Operands& o, int kernel, bool gate);
    hipError_t launch_mxfp4_tiles(hipStream_t s, const mx::Operands& o, int kernel, bool gate);
} // namespace nnf
