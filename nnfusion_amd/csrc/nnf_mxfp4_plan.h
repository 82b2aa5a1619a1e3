// Which kernel serves an MXFP4 product: shared by the library and the emitters (host arithmetic only).
#pragma once

#include <stddef.h>

namespace nnf
{
    namespace mx
    {
        constexpr int MAX_K = 1 << 22; // byte offsets inside a tile of 256 rows stay below 2^31
        // bytes from one row of scale bytes to the next: K / 32 rounded up to 16, so that every row starts on 16 bytes
        constexpr int scale_bytes(int K) { return ((K >> 5) + 15) & ~15; }
        constexpr bool supported(int K) { return K > 0 && K % 32 == 0 && K <= MAX_K; }

        // blocks of `rows` rows that there are at most, of M rows in `experts` groups (0: one product): every group may end in a block of its
        // own, which has a row at least
        constexpr long long most_row_blocks(int M, int experts, int rows)
        {
            const long long groups = experts == 0 ? 1 : experts < M ? experts : M;
            return (M + groups * (rows - 1)) / rows;
        }
        // tiles of columns of Y, `cols` weight rows each
        constexpr int column_tiles(int N, int cols, bool gate) { return (int)(((long long)N + (gate ? cols / 2 : cols) - 1) / (gate ? cols / 2 : cols)); }

        // a grid has fewer than 2^32 threads.  Of the products' kernels none has more than 512 in a workgroup
        constexpr long long MAX_WORKGROUPS = (1 << 23) - 1;
        // quantising and reading back take units of 512 values of a row, 16 of them to a workgroup of 256 threads
        constexpr int row_units(int K) { return (K + 511) / 512; }
        constexpr bool convertible(int rows, int K) { return (long long)rows * row_units(K) <= (1 << 28) - 16; }

        // activation rows x weight rows of a workgroup's tile.  DEEP: more steps of K under way, fewer wavefronts or workgroups a CU
        enum Kernel
        {
            ROWS_16x16, // operands straight into registers, eight ranges of K
            ROWS_16x32, // four
            TILE_8x32,  // through LDS, a wavefront for each range of K: four
            TILE_16x32, // eight
            TILE_16x64, // two
            TILE_16x64_DEEP, // one
            TILE_32x64, // four
            TILE_64x64, // four
            TILE_64x64_DEEP, // through LDS, the wavefronts share the tile and all of K
            TILE_128x128,
            TILE_128x128_DEEP,
            TILE_256x256,
            KERNELS
        };

        // What is known of a kernel: its tile, ranges of K, workgroups that a CU holds at once, values of a step of K, whether it has a
        // form with SiLU-gate, and the constants of its time in us,
        //   start + turn * (rounds - 1) + max(step * workgroups of a CU * steps, wait * rounds * steps) * (1 + off)
        // with the rounds of workgroups that a CU runs and `off` where rows of codes do not start on lines of memory (K no multiple of
        // 256).  Fitted to 6700 timings on one MI355X (weights read from HBM: 16 matrices from 512 x 2048 to 22016 x 4096 and 8192 x 8192
        // with 1 .. 4096 rows, nine mixtures of 4 .. 128 experts with 4 .. 16384 rows, even and uneven, each with and without SiLU-gate): 15 .. 24 %
        // (rms) from each; what they choose takes 1.02 (one matrix) and 1.03 (a mixture) times as long as the best of the kernels on
        // average, at most 1.5 times (12288 x 1056 with 24 .. 64 rows).
        struct KernelFacts
        {
            int rows, cols, ranges, per_cu, step_values;
            bool gate;
            float start, turn, step, wait, off;
        };
        constexpr KernelFacts FACTS[KERNELS] = {
            // (behind each: a product at which it is the fastest, its time and that of the next)
            {16, 16, 8, 3, 128, false, 2.80f, 1.11f, 0.465f, 0.607f, 0.00f},   // ROWS_16x16: 1 row by 4096 x 11008 in 8.2 us, the next best 10.5
            {16, 32, 4, 5, 128, true, 2.82f, 0.87f, 0.388f, 0.331f, 0.00f},    // ROWS_16x32: 64 rows, 60 experts of 2050 x 1376: 15.6 us, 20.9
            {8, 32, 4, 2, 256, false, 3.83f, 1.64f, 0.404f, 0.422f, 0.22f},    // TILE_8x32: 8 rows by 8192 x 8192: 9.8 us, 10.7
            {16, 32, 8, 1, 256, false, 3.49f, 2.02f, 1.117f, 1.137f, 0.07f},   // TILE_16x32: 128 rows by 1024 x 8192: 6.7 us, 8.6
            {16, 64, 2, 2, 256, true, 4.14f, 2.14f, 0.404f, 0.424f, 0.27f},    // TILE_16x64: 64 rows by 4096 x 11008: 13.9 us, 17.2
            {16, 64, 1, 2, 256, true, 4.06f, 2.64f, 0.226f, 0.355f, 0.18f},    // TILE_16x64_DEEP: 16 rows by 22016 x 4096: 12.6 us, 13.7
            {32, 64, 4, 1, 256, true, 3.69f, 2.46f, 0.293f, 1.012f, 0.13f},    // TILE_32x64: 64 rows by 8192 x 8192: 13.2 us, 16.3
            {64, 64, 4, 1, 256, true, 4.71f, 3.33f, 0.732f, 1.143f, 0.18f},    // TILE_64x64: 512 rows by 1024 x 8192: 11.3 us, 13.2
            {64, 64, 1, 2, 256, false, 3.95f, 1.98f, 0.291f, 0.305f, 0.16f},   // TILE_64x64_DEEP: 512 rows by 2050 x 2080: 11.2 us, 15.0
            {128, 128, 1, 2, 256, true, 4.58f, 4.87f, 0.678f, 0.808f, 0.12f},  // TILE_128x128: 4096 rows, 60 experts of 2050 x 1376: 43.6 us, 55.4
            {128, 128, 1, 1, 256, true, 5.22f, 5.03f, 0.566f, 0.637f, 0.21f},  // TILE_128x128_DEEP: 1024 rows by 4096 x 11008: 36.7 us, 48.5
            {256, 256, 1, 1, 256, true, 7.57f, 14.47f, 0.148f, 1.449f, 0.13f}, // TILE_256x256: 2048 rows by 8192 x 8192: 68.8 us, 93.6
        };

        // estimated time; experts == 0: one product, else M rows in that many groups, whose sizes are not known here
        inline float estimate(const KernelFacts& k, int M, int N, int K, bool gate, int experts, int num_cu)
        {
            // blocks of rows: a group ends in a block that is half full on average, and groups are of about one size
            float blocks = (float)((M + k.rows - 1) / k.rows);
            if (experts > 0)
            {
                const int groups = experts < M ? experts : M;
                blocks = groups * ((float)M / groups / k.rows + 0.5f);
                if (blocks < groups)
                    blocks = groups;
            }
            const int all_steps = (K + k.step_values - 1) / k.step_values;
            int steps = (all_steps + k.ranges - 1) / k.ranges;
            if (k.step_values == 256 && k.ranges > 1)
            {
                steps = (steps + 1) & ~1;
                if (steps > all_steps)
                    steps = all_steps;
            }
            const float a_cu = blocks * column_tiles(N, k.cols, gate) / num_cu;
            const float most = (float)(int)(a_cu + 0.99999f), rounds = (float)(int)((most + k.per_cu - 1) / k.per_cu);
            const float work = most * steps * k.step, wait = rounds * steps * k.wait;
            return (float)(k.start + k.turn * (rounds - 1) + (work > wait ? work : wait) * (K % 256 ? 1 + k.off : 1));
        }

        // whether a kernel has this form, in a grid that there can be
        constexpr bool fits(const KernelFacts& k, int M, int N, bool gate, int experts)
        {
            return (!gate || k.gate) && most_row_blocks(M, experts, k.rows) * column_tiles(N, k.cols, gate) <= MAX_WORKGROUPS;
        }

        // the kernel with the lowest estimate of those that fit; KERNELS: none does
        inline Kernel choose(int M, int N, int K, bool gate, int experts, int num_cu)
        {
            int best = KERNELS;
            float time = 0;
            for (int k = 0; k < KERNELS; ++k)
            {
                if (!fits(FACTS[k], M, N, gate, experts))
                    continue;
                const float t = estimate(FACTS[k], M, N, K, gate, experts, num_cu);
                if (best == KERNELS || t < time)
                    best = k, time = t;
            }
            return (Kernel)best;
        }
    } // namespace mx
} // namespace nnf
