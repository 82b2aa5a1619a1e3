// What the kernels on block-scaled 8-bit floating point share: their operands and the way of a sum into memory.
//
// A value is E4M3 (sign, four exponent bits, three mantissa bits; largest 448, no infinities); 128 values along K share an fp32 scale, in a
// weight matrix those of 128 rows too.
#pragma once

#include "../nnf_fp8_plan.h"
#include "grouped_tiles.h"
#include "nnf_device.h"

namespace nnf
{
    typedef __bf16 bf16_t;

    namespace fp8
    {
        typedef int intx8 __attribute__((ext_vector_type(8)));

        constexpr int E4M3 = 0; // operand format of the MFMA

        // Y[m, n] = sum over blocks b of K of As[b, m] Ws[n / 128, b] sum_k in b A[m, k] W[n, k]; with `offsets` the rows of A and Y are sorted by
        // expert: group e is the rows [offsets[e], offsets[e + 1]) and has the e-th of `experts` weight matrices
        struct Operands
        {
            const uint8_t* A;
            const float* As; // [blocks of K, M]
            const uint8_t* W;
            const float* Ws; // [blocks of N, blocks of K]; with SiLU-gate the gate rows' blocks, then the up rows'
            void* Y;
            const void* bias;     // [N] or null
            const void* residual; // [M, N] or null; may be Y
            const int* offsets;   // [experts + 1] or null
            int M, N, K;          // N columns of Y (with SiLU-gate 2 N weight rows: gate rows, then up rows)
            int experts;
            int bf16; // the type of Y, bias and residual: bf16, or fp16
        };

        // 32 values as an operand of the MFMA
        __device__ __forceinline__ intx8 operand(uintx4 a, uintx4 b)
        {
            return __builtin_shufflevector(__builtin_bit_cast(intx4, a), __builtin_bit_cast(intx4, b), 0, 1, 2, 3, 4, 5, 6, 7);
        }
    } // namespace fp8
} // namespace nnf
