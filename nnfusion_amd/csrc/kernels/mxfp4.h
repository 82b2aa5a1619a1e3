// What the kernels on microscaled 4-bit numbers (MXFP4) share: their operands.
//
// A value is E2M1 (sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), two to a byte with the even k in the low
// nibble; 32 values along K share the factor 2^(byte - 127), byte 255 standing for NaN (the OCP microscaling format).
#pragma once

#include "../nnf_mxfp4_plan.h"
#include "grouped_tiles.h"
#include "nnf_device.h"

namespace nnf
{
    namespace mx
    {
        typedef int intx8 __attribute__((ext_vector_type(8)));

        constexpr int FP4 = 4;        // operand format of the scaled MFMA
        constexpr uint32_t ONES = 0x7F7F7F7Fu; // four scale bytes of 2^0

        // Y[m, n] = sum_k A[m, k] W[n, k]; with `offsets` the rows of A and Y are sorted by expert: group e is the rows
        // [offsets[e], offsets[e + 1]) and has the e-th of `experts` weight matrices
        struct Operands
        {
            const uint8_t* A;
            const uint8_t* As;
            const uint8_t* W;
            const uint8_t* Ws;
            half_t* Y;
            const half_t* bias;     // [N] or null
            const half_t* residual; // [M, N] or null; may be Y
            const int* offsets;     // [experts + 1] or null
            int M, N, K;            // N columns of Y (with SiLU-gate 2 N weight rows: gate rows, then up rows)
            int experts;
        };

        // 32 four-bit values as an operand of the scaled MFMA, which reads the first four registers of this format
        __device__ __forceinline__ intx8 operand(uintx4 v)
        {
            const intx4 i = __builtin_bit_cast(intx4, v);
            return __builtin_shufflevector(i, i, 0, 1, 2, 3, -1, -1, -1, -1);
        }
    } // namespace mx
} // namespace nnf
