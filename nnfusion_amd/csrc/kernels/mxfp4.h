// What the kernels on microscaled 4-bit numbers (MXFP4) share: their operands, the search for a group of rows, the tail of a row.
//
// A value is E2M1 (sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), two to a byte with the even k in the low
// nibble; 32 values along K share the factor 2^(byte - 127), byte 255 standing for NaN (the OCP microscaling format).
#pragma once

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

        // `b`-th block of `1 << shift` rows: of all rows, or counted over the groups one after the other.  Every wavefront looks for
        // itself: 64 groups a turn, their numbers of blocks added up across the lanes.  Offsets are clamped to the rows there are, so
        // that no content of theirs leads outside the operands.  false: there is no such block.
        struct RowBlock
        {
            int expert, first, end; // rows [first, end) of the group from the block's first row on
        };
        __device__ __forceinline__ bool find_rows(const Operands& o, int b, int shift, RowBlock& found)
        {
            if (!o.offsets)
            {
                found = {0, b << shift, o.M};
                return (b << shift) < o.M;
            }
            const int lane = threadIdx.x & (WAVE - 1);
            for (int e0 = 0; e0 < o.experts; e0 += WAVE)
            {
                int first = 0, end = 0;
                if (e0 + lane < o.experts)
                {
                    first = min(max(o.offsets[e0 + lane], 0), o.M);
                    end = min(max(o.offsets[e0 + lane + 1], first), o.M);
                }
                const int blocks = (end - first + (1 << shift) - 1) >> shift;
                int sum = blocks;
#pragma unroll
                for (int d = 1; d < WAVE; d <<= 1)
                {
                    const int v = __shfl_up(sum, d, WAVE);
                    sum += lane >= d ? v : 0;
                }
                const uint64_t past = __ballot(sum > b);
                if (past)
                {
                    const int at = __builtin_ctzll(past);
                    found.expert = e0 + at;
                    found.first = __builtin_amdgcn_readlane(first, at) + ((b - (__builtin_amdgcn_readlane(sum, at) - __builtin_amdgcn_readlane(blocks, at))) << shift);
                    found.end = __builtin_amdgcn_readlane(end, at);
                    return true;
                }
                b -= __builtin_amdgcn_readlane(sum, WAVE - 1);
            }
            return false;
        }

        // bytes from one row of scale bytes to the next: K / 32 rounded up to 16, so that every row starts on 16 bytes
        __host__ __device__ __forceinline__ constexpr int mx_scale_stride(int K) { return ((K >> 5) + 15) & ~15; }

        // 32 four-bit values as an operand of the scaled MFMA, which reads the first four registers of this format
        __device__ __forceinline__ intx8 operand(uintx4 v)
        {
            const intx4 i = __builtin_bit_cast(intx4, v);
            return __builtin_shufflevector(i, i, 0, 1, 2, 3, -1, -1, -1, -1);
        }

        // position `id` of a grid of `n` workgroups -> the tile it takes.  Workgroups go to the eight XCDs in turn: this way each XCD, which
        // has an L2 of its own, works on one run of neighbouring tiles.
        __device__ __forceinline__ int xcd_order(int id, int n)
        {
            const int xcd = id & 7, each = n >> 3, more = n & 7;
            return xcd * each + min(xcd, more) + (id >> 3);
        }

        // bias and residual of four columns whose rows start on eight bytes
        __device__ __forceinline__ void add_four(const Operands& o, floatx4& y, int m, int n)
        {
            if (o.bias)
            {
                const half4_t v = *reinterpret_cast<const half4_t*>(o.bias + n);
                y += floatx4{(float)v.x, (float)v.y, (float)v.z, (float)v.w};
            }
            if (o.residual)
            {
                const half4_t v = *reinterpret_cast<const half4_t*>(o.residual + (size_t)m * o.N + n);
                y += floatx4{(float)v.x, (float)v.y, (float)v.z, (float)v.w};
            }
        }

        // Y[m, n .. n + 3] from fp32: bias and residual added in fp32, one rounding
        __device__ __forceinline__ void write_four(const Operands& o, floatx4 y, int m, int n)
        {
            const size_t at = (size_t)m * o.N + n;
            if ((o.N & 3) == 0)
            {
                if (n >= o.N)
                    return;
                add_four(o, y, m, n);
                *reinterpret_cast<half4_t*>(o.Y + at) = half4_t{(half_t)y.x, (half_t)y.y, (half_t)y.z, (half_t)y.w};
                return;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < o.N)
                {
                    float v = y[i];
                    if (o.bias)
                        v += (float)o.bias[n + i];
                    if (o.residual)
                        v += (float)o.residual[at + i];
                    o.Y[at + i] = (half_t)v;
                }
        }

        // Y[m, n .. n + 7], n a multiple of 8 below N
        __device__ __forceinline__ void write_eight(const Operands& o, floatx4 y0, floatx4 y1, int m, int n)
        {
            if (o.N & 7)
            {
                write_four(o, y0, m, n);
                write_four(o, y1, m, n + 4);
                return;
            }
            add_four(o, y0, m, n);
            add_four(o, y1, m, n + 4);
            *reinterpret_cast<half8_t*>(o.Y + (size_t)m * o.N + n) = half8_t{(half_t)y0.x, (half_t)y0.y, (half_t)y0.z, (half_t)y0.w,
                                                                             (half_t)y1.x, (half_t)y1.y, (half_t)y1.z, (half_t)y1.w};
        }

        // SiLU(g) * u in fp32
        __device__ __forceinline__ float silu_gate(float g, float u) { return g * (1.0f / (1.0f + __expf(-g))) * u; }
    } // namespace mx
} // namespace nnf
