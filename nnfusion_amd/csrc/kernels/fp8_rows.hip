// Block-scaled E4M3 x E4M3 for a few rows: the weights are read once, straight into the operand registers of the MFMA.
//
// A workgroup has 16 T weight rows (with SiLU-gate 16 T gate rows and their up rows) and a block of 16 activation rows; its W
// wavefronts cut K into as many ranges, each with the whole tile's sums in registers, which meet in LDS at the end.
// v_mfma_f32_16x16x128: lane l holds 32 values of row l % 16, the (l / 16)-th quarter of a block of K, so that a step's two loads of 16 bytes a lane
// take a whole line of each of 16 rows.  Its products are added to the sums times the activation row's and the weight block's scale.  The weights are
// the A operand: a lane has four consecutive columns of one row of Y, and their scale is one number a lane.  How exact the sums are: as in fp8_tile.hip.
//
// Bound by the latency of a batch of loads where a workgroup has few of them (one row by 4096 x 4096, 16.8 MB: 5.4 us, of which a launch takes
// 1.8; through LDS 6.6), else by HBM: 64 rows in 32 groups by 2048 x 4096, 268 MB, in 46 .. 47 us (5.7 TB/s; through LDS 52), with SiLU-gate, 537 MB, in 89
// (6.0 TB/s; 98); where 23, 24 and 27 of the 32 groups have rows in 69, 71 .. 74 and 80 (5.6 TB/s).  Every workgroup reads the activations
// anew, a line of each row for every 16 or 32 of weights: 16 rows by 11008 x 4096 take 13.7 us, 11.6 through LDS, one row 10.0.  Eight ranges of K in the place of
// four: 5.3 us for the first, 1.001 times the time of the best kernel on average where they are missing, so they are.
#include "fp8_launch.h"
#include "nnf_launch.h"

namespace nnf
{
    namespace
    {
        using namespace fp8;

        constexpr int ROWS = 16, W = 4; // activation rows of a workgroup, its wavefronts

        // T tiles of 16 weight rows
        template <int T, bool GATE>
        __global__ __launch_bounds__(W* WAVE) void fp8_rows_kernel(Operands o, int col_tiles)
        {
            constexpr int TW = GATE ? 2 * T : T, NS = GATE ? 2 : 1; // tiles of weight rows, scales of the weights
            constexpr int BATCH = 4;                                // steps whose loads are under way together
            __shared__ floatx4 parts[W][TW][WAVE];
            const int lane = threadIdx.x & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
            TileAt rows;
            if (!find_tile(o, blockIdx.x, ROWS, col_tiles, rows))
                return;
            const int n0 = rows.column * (16 * T);
            const int r = lane & 15, g = lane >> 4;
            const int row_bytes = o.K, steps = blocks_of(o.K), part = (steps + W - 1) / W, end = min(steps, (wave + 1) * part);

            // rows past the end repeat the last one: their results are not written
            const uint8_t* const w_base = o.W + ((size_t)rows.expert * (GATE ? 2 * (size_t)o.N : o.N) + n0) * row_bytes;
            const uint8_t* const a_base = o.A + (size_t)rows.first * row_bytes;
            const int a_row = min(r, rows.end - rows.first - 1), n_blocks = blocks_of(o.N);
            const float* const as_base = o.As + (rows.first + a_row);
            const float* const ws_base = o.Ws + ((size_t)rows.expert * (NS * n_blocks) + n0 / BLOCK) * steps;
            uint32_t w[TW];
#pragma unroll
            for (int t = 0; t < TW; ++t)
                w[t] = (uint32_t)(min((t % T) * 16 + r, o.N - 1 - n0) + (t >= T ? o.N : 0)) * row_bytes + g * 32;
            const uint32_t a = (uint32_t)a_row * row_bytes + g * 32;

            floatx4 sum[TW] = {};
            // `count` steps from `step` on.  LAST: the last of them may end behind the rows: there a lane reads the step's first piece, and the
            // weights count as zeros (the activations repeat values of their row: NaN only in rows that are NaN anyway)
            const auto batch = [&](int step, auto count, auto last) {
                constexpr int C = count;
                uintx4 wv[TW][C][2], av[C][2];
                float as[C], ws[NS][C];
                const int left = row_bytes - (step + C - 1) * BLOCK; // of the last step
#pragma unroll
                for (int s = 0; s < C; ++s)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                    {
                        const int at = h * 16 - (last && s == C - 1 && g * 32 + h * 16 >= left ? g * 32 + h * 16 : 0);
#pragma unroll
                        for (int t = 0; t < TW; ++t)
                            wv[t][s][h] = *reinterpret_cast<const uintx4*>(w_base + (step + s) * BLOCK + (w[t] + at));
                        av[s][h] = *reinterpret_cast<const uintx4*>(a_base + (step + s) * BLOCK + (a + at));
                    }
#pragma unroll
                for (int s = 0; s < C; ++s)
                {
                    as[s] = as_base[(size_t)(step + s) * o.M];
#pragma unroll
                    for (int i = 0; i < NS; ++i)
                        ws[i][s] = ws_base[(size_t)i * n_blocks * steps + step + s];
                }
                if constexpr (last)
#pragma unroll
                    for (int t = 0; t < TW; ++t)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            wv[t][C - 1][h] = g * 32 + h * 16 < left ? wv[t][C - 1][h] : uintx4{0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < C; ++s)
#pragma unroll
                    for (int t = 0; t < TW; ++t)
                    {
                        const floatx4 product = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(wv[t][s][0], wv[t][s][1]), operand(av[s][0], av[s][1]), floatx4{}, E4M3,
                                                                                                 E4M3, 0, 0, 0, 0);
                        const float scale = as[s] * ws[t / T][s];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            sum[t][i] = __builtin_fmaf(product[i], scale, sum[t][i]);
                    }
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
                    o.bf16 ? write_four<bf16_t>(o, y, m, n0 + f * 16 + g * 4) : write_four<half_t>(o, y, m, n0 + f * 16 + g * 4);
            }
        }

        template <int T, bool GATE>
        hipError_t launch(hipStream_t s, const Operands& o)
        {
            const int col_tiles = tiles_of_columns(FACTS[T == 1 ? ROWS_16x16 : ROWS_16x32], o.N, GATE);
            fp8_rows_kernel<T, GATE><<<(unsigned)(row_blocks(o, ROWS) * col_tiles), W * WAVE, 0, s>>>(o, col_tiles);
            return hipGetLastError();
        }
    } // namespace

    hipError_t launch_fp8_rows(hipStream_t s, const fp8::Operands& o, int kernel, bool gate)
    {
        switch (kernel)
        {
        case fp8::ROWS_16x16: return gate ? launch<1, true>(s, o) : launch<1, false>(s, o);
        default: return gate ? launch<2, true>(s, o) : launch<2, false>(s, o);
        }
    }
} // namespace nnf
