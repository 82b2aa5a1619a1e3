// What the kernels on microscaled 4-bit numbers (MXFP4) share: their operands, the search for a group of rows, the tail of a row.
//
// A value is E2M1 (sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), two to a byte with the even k in the low
// nibble; 32 values along K share the factor 2^(byte - 127), byte 255 standing for NaN (the OCP microscaling format).
#pragma once

#include "../nnf_mxfp4_plan.h"
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

        inline long long row_blocks(const Operands& o, int rows) { return most_row_blocks(o.M, o.offsets ? o.experts : 0, rows); }

        // The tile that workgroup `id` takes, of a product in blocks of `rows` rows and `col_tiles` tiles of columns: the groups one
        // after the other; inside a group up to GROUPED row blocks of one column one after the other, then the next column, so that
        // neighbours share their weights and the few rows of activations.  Workgroups go to the eight XCDs in turn, each of which has an
        // L2 of its own: the order of the tiles is cut into eight runs, one an XCD.  Every wavefront looks for itself: 64 groups a turn, their
        // numbers of blocks added up across the lanes.  Offsets are clamped to the rows there are, so that no content of theirs leads
        // outside the operands.  false: there are no more tiles.
        constexpr int GROUPED = 8;
        struct TileAt
        {
            int expert, first, end; // rows [first, end) of the group from the tile's first row on
            int column;             // tile of columns
        };
        __device__ __forceinline__ int xcd_order(int id, int n)
        {
            const int xcd = id & 7, each = n >> 3, more = n & 7;
            return xcd * each + min(xcd, more) + (id >> 3);
        }
        // rows [first, end) of the lane's group and its number of blocks
        __device__ __forceinline__ int group_of_lane(const Operands& o, int e, int rows, int& first, int& end)
        {
            first = 0, end = 0;
            if (e < o.experts)
            {
                first = min(max(o.offsets[e], 0), o.M);
                end = min(max(o.offsets[e + 1], first), o.M);
            }
            return (end - first + rows - 1) / rows;
        }
        // sum over the lanes 0 .. own, in each lane: four shifts inside the rows of 16 lanes, then the rows' last lanes passed on
        __device__ __forceinline__ int sum_up_to_lane(int v)
        {
            v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false); // row_shr:1
            v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false); // row_shr:2
            v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false); // row_shr:4
            v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false); // row_shr:8
            v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false); // row_bcast:15 into rows 1 and 3
            v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false); // row_bcast:31 into rows 2 and 3
            return v;
        }
        __device__ __forceinline__ bool find_tile(const Operands& o, int id, int rows, int col_tiles, TileAt& found)
        {
            int begin = 0, end = o.M, blocks = (o.M + rows - 1) / rows, expert = 0;
            if (!o.offsets)
            {
                if (id >= blocks * col_tiles)
                    return false;
                id = xcd_order(id, blocks * col_tiles);
            }
            else
            {
                const int lane = threadIdx.x & (WAVE - 1);
                int first, last, own = group_of_lane(o, lane, rows, first, last), sum = sum_up_to_lane(own);
                int all = __builtin_amdgcn_readlane(sum, WAVE - 1);
                for (int e0 = WAVE; e0 < o.experts; e0 += WAVE)
                {
                    int f, l;
                    all += __builtin_amdgcn_readlane(sum_up_to_lane(group_of_lane(o, e0 + lane, rows, f, l)), WAVE - 1);
                }
                if (id >= all * col_tiles)
                    return false;
                id = xcd_order(id, all * col_tiles);
                // the block that the tile would have if a block's columns came one after the other: it is of the same group
                const int b = id / col_tiles;
                int before = 0;
                while (b >= before + __builtin_amdgcn_readlane(sum, WAVE - 1))
                {
                    before += __builtin_amdgcn_readlane(sum, WAVE - 1);
                    expert += WAVE;
                    if (expert >= o.experts)
                        return false; // (offsets that overlap may count more blocks than an int holds)
                    own = group_of_lane(o, expert + lane, rows, first, last);
                    sum = sum_up_to_lane(own);
                }
                const uint64_t past = __ballot(before + sum > b);
                const int at = past ? __builtin_ctzll(past) : 0;
                blocks = __builtin_amdgcn_readlane(own, at);
                id -= (before + __builtin_amdgcn_readlane(sum, at) - blocks) * col_tiles;
                begin = __builtin_amdgcn_readlane(first, at);
                end = __builtin_amdgcn_readlane(last, at);
                expert += at;
                if ((unsigned)id >= (unsigned)(blocks * col_tiles))
                    return false;
            }
            const int g = id / (GROUPED * col_tiles), of_group = min(blocks - g * GROUPED, GROUPED);
            id -= g * (GROUPED * col_tiles);
            const int column = id / of_group, block = g * GROUPED + id - column * of_group;
            found = {expert, begin + block * rows, end, column};
            return true;
        }

        // 32 four-bit values as an operand of the scaled MFMA, which reads the first four registers of this format
        __device__ __forceinline__ intx8 operand(uintx4 v)
        {
            const intx4 i = __builtin_bit_cast(intx4, v);
            return __builtin_shufflevector(i, i, 0, 1, 2, 3, -1, -1, -1, -1);
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

        // Y[row(i), n .. n + 7] for each i with a row (row(i) < 0: none), n a multiple of 8 below N
        template <int COUNT, class Row>
        __device__ __forceinline__ void write_rows(const Operands& o, floatx4 (&y)[COUNT][2], int n, Row row)
        {
            if (o.N & 7)
            {
#pragma unroll
                for (int i = 0; i < COUNT; ++i)
                    if (row(i) >= 0)
                    {
                        write_four(o, y[i][0], row(i), n);
                        write_four(o, y[i][1], row(i), n + 4);
                    }
                return;
            }
            if (o.bias)
            {
                const half8_t v = *reinterpret_cast<const half8_t*>(o.bias + n);
#pragma unroll
                for (int i = 0; i < COUNT; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        y[i][e / 4][e % 4] += (float)v[e];
            }
            if (o.residual)
            {
                half8_t v[COUNT];
#pragma unroll
                for (int i = 0; i < COUNT; ++i)
                    v[i] = *reinterpret_cast<const half8_t*>(o.residual + (size_t)max(row(i), 0) * o.N + n);
#pragma unroll
                for (int i = 0; i < COUNT; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        y[i][e / 4][e % 4] += (float)v[i][e];
            }
#pragma unroll
            for (int i = 0; i < COUNT; ++i)
                if (row(i) >= 0)
                    *reinterpret_cast<half8_t*>(o.Y + (size_t)row(i) * o.N + n) = half8_t{(half_t)y[i][0].x, (half_t)y[i][0].y, (half_t)y[i][0].z, (half_t)y[i][0].w,
                                                                                         (half_t)y[i][1].x, (half_t)y[i][1].y, (half_t)y[i][1].z, (half_t)y[i][1].w};
        }

        // SiLU(g) * u in fp32
        __device__ __forceinline__ float silu_gate(float g, float u) { return g * (1.0f / (1.0f + __expf(-g))) * u; }
    } // namespace mx
} // namespace nnf
