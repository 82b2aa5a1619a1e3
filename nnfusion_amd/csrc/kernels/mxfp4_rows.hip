// MXFP4 x MXFP4 for a few rows: the weights are read once, straight into the operand registers of the MFMA.
//
// A workgroup has 16 T weight rows (with SiLU-gate 16 T gate rows and their up rows) and a block of 16 B activation rows; its
// wavefronts split K into units of 512 values, dealt out in turn, each with the whole tile's sums in registers, which meet in LDS at
// the end.  v_mfma_scale_f32_16x16x128: lane l holds 32 values of row l % 16, the (l / 16)-th block of the step's four, so a load
// of 16 bytes a lane covers 64 contiguous bytes of each of 16 rows; a row's 16 scale bytes of a unit are one load, from which each
// lane takes the byte of its block.  The weights are the A operand: a lane then has four consecutive columns of one row of Y.
#include "mxfp4.h"
#include "mxfp4_launch.h"
#include "nnf_launch.h"

namespace nnf
{
    namespace
    {
        using namespace mx;

        constexpr int UNIT_BYTES = 256; // of a row: 512 values

        // T tiles of 16 weight rows, B blocks of 16 activation rows, W wavefronts
        template <int T, int B, int W, bool GATE>
        __global__ __launch_bounds__(W* WAVE) void mxfp4_rows_kernel(Operands o, int col_tiles)
        {
            constexpr int TW = GATE ? 2 * T : T; // tiles of weight rows
            __shared__ floatx4 parts[W][TW * B][WAVE];
            const int lane = threadIdx.x & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
            RowBlock rows;
            constexpr int SHIFT = B == 1 ? 4 : B == 2 ? 5 : 6;
            const int block = blockIdx.x / col_tiles;
            if (!find_rows(o, block, SHIFT, rows))
                return;
            const int n0 = (blockIdx.x - block * col_tiles) * (16 * T);
            const int r = lane & 15, g = lane >> 4;
            const int row_bytes = o.K >> 1, scale_stride = mx_scale_stride(o.K);
            const int units = (o.K + 511) >> 9;

            // rows past the end repeat the last one: their results are not written
            const uint8_t *w[TW], *ws[TW], *a[B], *as[B];
#pragma unroll
            for (int t = 0; t < TW; ++t)
            {
                const size_t row = (size_t)rows.expert * (GATE ? 2 * o.N : o.N) + min(n0 + (t % T) * 16 + r, o.N - 1) + (t >= T ? o.N : 0);
                w[t] = o.W + row * row_bytes;
                ws[t] = o.Ws + row * scale_stride;
            }
#pragma unroll
            for (int b = 0; b < B; ++b)
            {
                const size_t row = min(rows.first + b * 16 + r, rows.end - 1);
                a[b] = o.A + row * row_bytes;
                as[b] = o.As + row * scale_stride;
            }

            floatx4 sum[TW][B] = {};
            for (int u = wave; u < units; u += W)
            {
                const bool whole = (u + 1) * UNIT_BYTES <= row_bytes;
                uintx4 wv[TW][4], av[B][4], wsv[TW], asv[B];
                int at[4];
#pragma unroll
                for (int s = 0; s < 4; ++s)
                {
                    at[s] = u * UNIT_BYTES + s * 64 + g * 16;
                    if (!whole)
                        at[s] = min(at[s], row_bytes - 16);
                }
#pragma unroll
                for (int t = 0; t < TW; ++t)
                {
                    wsv[t] = *reinterpret_cast<const uintx4*>(ws[t] + u * 16);
#pragma unroll
                    for (int s = 0; s < 4; ++s)
                        wv[t][s] = *reinterpret_cast<const uintx4*>(w[t] + at[s]);
                }
#pragma unroll
                for (int b = 0; b < B; ++b)
                {
                    asv[b] = *reinterpret_cast<const uintx4*>(as[b] + u * 16);
#pragma unroll
                    for (int s = 0; s < 4; ++s)
                        av[b][s] = *reinterpret_cast<const uintx4*>(a[b] + at[s]);
                }
                if (!whole)
                {
                    // blocks behind the end of a row: zeros times zeros, whatever stands there
#pragma unroll
                    for (int s = 0; s < 4; ++s)
                    {
                        const bool there = u * UNIT_BYTES + s * 64 + g * 16 < row_bytes;
#pragma unroll
                        for (int t = 0; t < TW; ++t)
                        {
                            wv[t][s] = there ? wv[t][s] : uintx4{0, 0, 0, 0};
                            wsv[t][s] = there ? wsv[t][s] : ONES;
                        }
#pragma unroll
                        for (int b = 0; b < B; ++b)
                            asv[b][s] = there ? asv[b][s] : ONES;
                    }
                }
#pragma unroll
                for (int s = 0; s < 4; ++s)
#pragma unroll
                    for (int t = 0; t < TW; ++t)
#pragma unroll
                        for (int b = 0; b < B; ++b)
                            sum[t][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(wv[t][s]), operand(av[b][s]), sum[t][b], FP4, FP4, 0,
                                                                                         (int)(wsv[t][s] >> (8 * g)), 0, (int)(asv[b][s] >> (8 * g)));
            }
#pragma unroll
            for (int t = 0; t < TW; ++t)
#pragma unroll
                for (int b = 0; b < B; ++b)
                    parts[wave][t * B + b][lane] = sum[t][b];
            __syncthreads();
            // the wavefronts' sums in the order of the wavefronts; fragment f of the tile to wavefront f mod W
            for (int f = wave; f < T * B; f += W)
            {
                floatx4 y = parts[0][f][lane];
                for (int i = 1; i < W; ++i)
                    y += parts[i][f][lane];
                if constexpr (GATE)
                {
                    floatx4 up = parts[0][T * B + f][lane];
                    for (int i = 1; i < W; ++i)
                        up += parts[i][T * B + f][lane];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        y[i] = silu_gate(y[i], up[i]);
                }
                const int m = rows.first + (f % B) * 16 + r;
                if (m < rows.end)
                    write_four(o, y, m, n0 + (f / B) * 16 + g * 4);
            }
        }

        template <int T, int B, int W, bool GATE>
        hipError_t launch(hipStream_t s, const Operands& o, int row_blocks)
        {
            const int col_tiles = (o.N + 16 * T - 1) / (16 * T);
            mxfp4_rows_kernel<T, B, W, GATE><<<(unsigned)row_blocks * col_tiles, W * WAVE, 0, s>>>(o, col_tiles);
            return hipGetLastError();
        }
    } // namespace

    hipError_t launch_mxfp4_rows(hipStream_t s, const mx::Operands& o, int row_shift, int row_blocks, bool gate)
    {
        if (gate)
            return row_shift == 4 ? launch<1, 1, 8, true>(s, o, row_blocks) : row_shift == 5 ? launch<1, 2, 8, true>(s, o, row_blocks) : launch<1, 4, 8, true>(s, o, row_blocks);
        return row_shift == 4 ? launch<1, 1, 8, false>(s, o, row_blocks) : row_shift == 5 ? launch<1, 2, 8, false>(s, o, row_blocks) : launch<2, 4, 8, false>(s, o, row_blocks);
    }
} // namespace nnf
