// MXFP4 x MXFP4 for a few rows: the weights are read once, straight into the operand registers of the MFMA.
//
// A workgroup has 16 T weight rows (with SiLU-gate 16 T gate rows and their up rows) and a block of 16 activation rows; its W
// wavefronts cut K into as many ranges, each with the whole tile's sums in registers, which meet in LDS at the end.
// v_mfma_scale_f32_16x16x128: lane l holds 32 values of row l % 16, the (l / 16)-th block of the step's four, so a load of 16 bytes a
// lane covers 64 contiguous bytes of each of 16 rows; the row's four scale bytes of the step are one word, from which each lane takes
// its own (the memory pipeline's time goes by the lines that a load touches: the words of four steps are one load).  The weights are the
// A operand: a lane then has four consecutive columns of one row of Y.
//
// Bound by the latency of a batch of loads where few workgroups have few batches (one row by 4096 x 4096, 8.9 MB: 4.2 us), then by the half
// lines that its loads take (16 rows by 12288 x 4096, 27 MB: 10.6 us; the tile kernel, which loads whole lines into LDS, 8.1).  It is the
// fastest where a row of K is a few steps or does not start on a line: 333 rows in 60 groups by 2050 x 1376, 57 MB, in 14 us, 19.7
// where the weights come from HBM (tiles through LDS: 22 and more).  92 registers instead of 104, for a fifth wavefront on a SIMD, changed
// nothing.
#include "mxfp4.h"
#include "mxfp4_launch.h"
#include "nnf_launch.h"

namespace nnf
{
    namespace
    {
        using namespace mx;

        constexpr int ROWS = 16; // activation rows of a workgroup
        typedef uintx4 words4 __attribute__((aligned(4))); // a load of 16 bytes that begins at any word

        // T tiles of 16 weight rows, W wavefronts
        template <int T, int W, bool GATE>
        __global__ __launch_bounds__(W* WAVE) void mxfp4_rows_kernel(Operands o, int col_tiles)
        {
            constexpr int TW = GATE ? 2 * T : T; // tiles of weight rows
            constexpr int BATCH = 4;             // steps whose loads are under way together
            __shared__ floatx4 parts[W][TW][WAVE];
            const int lane = threadIdx.x & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
            TileAt rows;
            if (!find_tile(o, blockIdx.x, ROWS, col_tiles, rows))
                return;
            const int n0 = rows.column * (16 * T);
            const int r = lane & 15, g = lane >> 4;
            const int row_bytes = o.K >> 1, scale_stride = scale_bytes(o.K);
            const int steps = (o.K + 127) >> 7, part = (steps + W - 1) / W, end = min(steps, (wave + 1) * part);

            // rows past the end repeat the last one: their results are not written
            const size_t w_row = (size_t)rows.expert * (GATE ? 2 * o.N : o.N) + n0;
            const uint8_t* const w_base = o.W + w_row * row_bytes;
            const uint8_t* const ws_base = o.Ws + w_row * scale_stride;
            const uint8_t* const a_base = o.A + (size_t)rows.first * row_bytes;
            const uint8_t* const as_base = o.As + (size_t)rows.first * scale_stride;
            uint32_t w[TW], ws[TW];
#pragma unroll
            for (int t = 0; t < TW; ++t)
            {
                const uint32_t row = min((t % T) * 16 + r, o.N - 1 - n0) + (t >= T ? o.N : 0);
                w[t] = row * row_bytes + g * 16;
                ws[t] = row * scale_stride;
            }
            const uint32_t a_row = min(r, rows.end - rows.first - 1), a = a_row * row_bytes + g * 16, as = a_row * scale_stride;

            floatx4 sum[TW] = {};
            // `count` steps from `step` on.  LAST: the last of them may end behind the rows: there a lane reads the first block of the step,
            // and the weights count as zeros, times 2^0 of both operands
            const auto batch = [&](int step, auto count, auto last) {
                constexpr int C = count;
                uintx4 wv[TW][C], av[C], wsv[TW], asv;
                const bool there = (step + C - 1) * 64 + g * 16 < row_bytes;
                const uint32_t back = last && !there ? g * 16 : 0; // bytes back to the first block
                // the scale bytes of the batch are one load of 16 bytes a row, as far as the row's (padded) end lets it begin there: `skip` words
                // of it belong to the steps before
                const int scale_from = min(step * 4, scale_stride - 16), skip = step - scale_from / 4;
#pragma unroll
                for (int t = 0; t < TW; ++t)
                    wsv[t] = *reinterpret_cast<const words4*>(ws_base + scale_from + ws[t]);
                asv = *reinterpret_cast<const words4*>(as_base + scale_from + as);
#pragma unroll
                for (int s = 0; s < C; ++s)
                {
#pragma unroll
                    for (int t = 0; t < TW; ++t)
                        wv[t][s] = *reinterpret_cast<const uintx4*>(w_base + (step + s) * 64 + (w[t] - (s == C - 1 ? back : 0)));
                    av[s] = *reinterpret_cast<const uintx4*>(a_base + (step + s) * 64 + (a - (s == C - 1 ? back : 0)));
                }
                if (skip)
                {
                    const auto moved = [&](uintx4 v) {
                        return skip == 1 ? uintx4{v.y, v.z, v.w, ONES} : skip == 2 ? uintx4{v.z, v.w, ONES, ONES} : uintx4{v.w, ONES, ONES, ONES};
                    };
#pragma unroll
                    for (int t = 0; t < TW; ++t)
                        wsv[t] = moved(wsv[t]);
                    asv = moved(asv);
                }
                if constexpr (last)
                {
#pragma unroll
                    for (int t = 0; t < TW; ++t)
                    {
                        wv[t][C - 1] = there ? wv[t][C - 1] : uintx4{0, 0, 0, 0};
                        wsv[t][C - 1] = there ? wsv[t][C - 1] : ONES;
                    }
                    asv[C - 1] = there ? asv[C - 1] : ONES;
                }
#pragma unroll
                for (int s = 0; s < C; ++s)
#pragma unroll
                    for (int t = 0; t < TW; ++t)
                        sum[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(wv[t][s]), operand(av[s]), sum[t], FP4, FP4, 0,
                                                                                  (int)(wsv[t][s] >> (8 * g)), 0, (int)(asv[s] >> (8 * g)));
            };
            int step = wave * part;
            for (; step + BATCH < end; step += BATCH)
                batch(step, std::integral_constant<int, BATCH>{}, std::false_type{});
            unroll_for<1, BATCH + 1>([&](auto c) {
                if (end - step == c)
                    batch(step, c, std::true_type{});
            });
#pragma unroll
            for (int t = 0; t < TW; ++t)
                parts[wave][t][lane] = sum[t];
            __syncthreads();
            // the wavefronts' sums in the order of the wavefronts; fragment f of the tile to wavefront f mod W
            for (int f = wave; f < T; f += W)
            {
                floatx4 y = parts[0][f][lane];
#pragma unroll
                for (int i = 1; i < W; ++i)
                    y += parts[i][f][lane];
                if constexpr (GATE)
                {
                    floatx4 up = parts[0][T + f][lane];
#pragma unroll
                    for (int i = 1; i < W; ++i)
                        up += parts[i][T + f][lane];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        y[i] = silu_gate(y[i], up[i]);
                }
                const int m = rows.first + r;
                if (m < rows.end)
                    write_four<half_t>(o, y, m, n0 + f * 16 + g * 4);
            }
        }

        template <int T, int W, bool GATE>
        hipError_t launch(hipStream_t s, const Operands& o)
        {
            const int col_tiles = column_tiles(o.N, (GATE ? 2 : 1) * 16 * T, GATE);
            mxfp4_rows_kernel<T, W, GATE><<<(unsigned)(row_blocks(o, ROWS) * col_tiles), W * WAVE, 0, s>>>(o, col_tiles);
            return hipGetLastError();
        }
    } // namespace

    hipError_t launch_mxfp4_rows(hipStream_t s, const mx::Operands& o, int kernel, bool gate)
    {
        if (gate)
            return launch<1, 4, true>(s, o); // a gate tile and its up tile: 16 x 32
        return kernel == mx::ROWS_16x16 ? launch<1, 8, false>(s, o) : launch<2, 4, false>(s, o);
    }
} // namespace nnf
