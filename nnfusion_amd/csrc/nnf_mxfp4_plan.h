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

        // sizes that a product may have.  With SiLU-gate the bytes from a gate row to its up row are counted in 32 bits
        constexpr bool product_supported(int M, int N, int K, bool gate)
        {
            return supported(K) && M <= 1 << 30 && N <= 1 << 29 && (!gate || (long long)N * K < 1LL << 32);
        }

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
            TILE_32x128, // through LDS, the wavefronts share the tile and all of K
            TILE_64x64_DEEP,
            TILE_64x128,
            TILE_64x128_DEEP,
            TILE_128x128,
            TILE_128x128_DEEP,
            TILE_256x256,
            KERNELS
        };

        // What is known of a kernel: its tile, ranges of K, workgroups that a CU holds at once, values of a step of K, whether it has a
        // form with SiLU-gate, and the constants of its time in us,
        //   start + turn * (rounds - 1) + max(step * workgroups of a CU * steps, wait * rounds * steps) * (1 + off)
        // with the rounds of workgroups that a CU runs and `off` where rows of codes do not start on lines of memory (K no multiple of
        // 256).  Fitted to 9800 timings on one MI355X (weights read from HBM: 16 matrices from 512 x 2048 to 22016 x 4096 and 8192 x 8192
        // with 1 .. 4096 rows, nine mixtures of 4 .. 128 experts with 4 .. 16384 rows, even and uneven, each with and without SiLU-gate), those
        // of the kernels near the fastest with more weight: 15 .. 24 % (rms) from each; what they choose takes 1.02 times as long as the best of
        // the kernels on average (matrices that the fit has not seen: 1.02, mixtures 1.03), at most 1.45 times (64 rows in 4 uneven
        // groups by 4096 x 11008).
        struct KernelFacts
        {
            int rows, cols, ranges, per_cu, step_values;
            bool gate;
            float start, turn, step, wait, off;
        };
        constexpr KernelFacts FACTS[KERNELS] = {
            // (behind each: a product at which it is the fastest, its time and that of the next)
            {16, 16, 8, 3, 128, false, 2.80f, 0.02f, 0.476f, 0.408f, 0.00f},   // ROWS_16x16: 1 row by 4096 x 11008 in 8.0 us, the next best 10.4
            {16, 32, 4, 5, 128, true, 2.64f, 0.01f, 0.334f, 0.414f, 0.00f},    // ROWS_16x32: 16 rows by 2050 x 2080, SiLU-gate: 4.4 us, 7.8
            {8, 32, 4, 2, 256, false, 3.42f, 1.23f, 0.453f, 0.357f, 0.31f},    // TILE_8x32: 8 rows by 8192 x 8192: 9.7 us, 10.7
            {16, 32, 8, 1, 256, false, 3.40f, 1.91f, 0.898f, 1.101f, 0.15f},   // TILE_16x32: 128 rows by 1024 x 8192: 6.4 us, 8.2
            {16, 64, 2, 2, 256, true, 4.02f, 1.86f, 0.411f, 0.336f, 0.30f},    // TILE_16x64: 48 rows by 4096 x 11008: 13.6 us, 16.5
            {16, 64, 1, 2, 256, true, 4.20f, 2.47f, 0.231f, 0.318f, 0.13f},    // TILE_16x64_DEEP: 64 rows, 4 experts of 4096 x 11008, SiLU-gate: 26.4 us, 28.2
            {32, 64, 4, 1, 256, true, 3.20f, 1.84f, 0.464f, 1.110f, 0.28f},    // TILE_32x64: 128 rows by 4096 x 4096, SiLU-gate: 6.9 us, 8.9
            {64, 64, 4, 1, 256, true, 4.49f, 2.59f, 0.884f, 1.290f, 0.22f},    // TILE_64x64: 128 rows by 8192 x 8192, SiLU-gate: 16.5 us, 22.0
            {32, 128, 1, 2, 256, false, 3.21f, 2.64f, 0.418f, 0.381f, 0.36f},  // TILE_32x128: 256 rows, 8 experts of 2048 x 4096: 10.1 us, 11.5
            {64, 64, 1, 2, 256, false, 3.90f, 1.78f, 0.296f, 0.277f, 0.31f},   // TILE_64x64_DEEP: 64 rows, 4 experts of 4096 x 11008: 22.7 us, 26.2
            {64, 128, 1, 2, 256, true, 3.42f, 3.60f, 0.545f, 0.706f, 0.13f},   // TILE_64x128: 1024 rows, 32 experts of 1024 x 1024, SiLU-gate: 8.4 us, 10.8
            {64, 128, 1, 1, 256, true, 4.72f, 3.83f, 0.467f, 0.467f, 0.14f},   // TILE_64x128_DEEP: 384 rows by 4096 x 11008, SiLU-gate: 27.0 us, 34.9
            {128, 128, 1, 2, 256, true, 4.75f, 5.28f, 0.620f, 0.827f, 0.17f},  // TILE_128x128: 4096 rows, 60 experts of 2050 x 1376, SiLU-gate: 40.6 us, 50.5
            {128, 128, 1, 1, 256, true, 5.31f, 4.68f, 0.593f, 0.640f, 0.27f},  // TILE_128x128_DEEP: 1024 rows by 4096 x 11008: 37.0 us, 48.1
            {256, 256, 1, 1, 256, true, 7.30f, 12.58f, 1.145f, 1.538f, 0.19f}, // TILE_256x256: 2048 rows by 8192 x 8192: 66.7 us, 89.2
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
            // (unrolled: divisions by constants, 0.12 us in place of 0.33)
#pragma GCC unroll 16
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
