// Which kernel serves an MXFP4 product: shared by the library and the emitters (host arithmetic only).
#pragma once

#include "nnf_tiles_plan.h"

#include <stddef.h>

namespace nnf
{
    namespace mx
    {
        using nnf::column_tiles;
        using nnf::most_row_blocks;

        constexpr int MAX_K = 1 << 22; // byte offsets inside a tile of 256 rows stay below 2^31
        // bytes from one row of scale bytes to the next: K / 32 rounded up to 16, so that every row starts on 16 bytes
        constexpr int scale_bytes(int K) { return ((K >> 5) + 15) & ~15; }
        constexpr bool supported(int K) { return K > 0 && K % 32 == 0 && K <= MAX_K; }

        // sizes that a product may have (experts == 0: one weight matrix).  With SiLU-gate the bytes from a gate row to its up row are counted
        // in 32 bits; groups are looked through 64 at a time, and the first number behind them is an int too
        constexpr bool product_supported(int M, int N, int K, bool gate, int experts)
        {
            return supported(K) && M <= 1 << 30 && N <= 1 << 29 && (!gate || (long long)N * K < 1LL << 32) && experts <= 1 << 30;
        }

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
            TILE_8x32,  // through LDS, a wavefront for each range of K: two
            TILE_16x32, // one
            TILE_16x32_2, // two
            TILE_16x32_4, // four
            TILE_16x64, // two
            TILE_32x64, // four
            TILE_32x128, // through LDS, the wavefronts share the tile and all of K
            TILE_64x64,
            TILE_64x128,
            TILE_64x128_DEEP,
            TILE_128x128,
            TILE_128x128_DEEP,
            TILE_256x256,
            KERNELS
        };

        // What is known of a kernel: its tile, ranges of K, workgroups that a CU holds at once, values of a step of K, whether it has a
        // form with SiLU-gate, and the constants of its time in us,
        //   start + turn * (rounds - 1) + max(step * workgroups of a CU * steps * (1 + off), wait * rounds * steps * (1 + off), bytes / rate)
        // with the rounds of workgroups that a CU runs and `off` where rows of codes do not start on lines of memory (K no multiple of
        // 256).  `rate` is a constant of the fit as the others are, in TB/s, and not the memory's (a plain read of 1 GiB reaches 6.2): of a
        // mixture every group's matrix counts, also those that no row goes to, and small products come from the caches in part.  Held
        // below 6, the fit chooses worse: 1.03 times the best on average in place of 1.02.
        //
        // Fitted to 16900 timings on one MI355X (weights read from HBM: 19 matrices from 512 x 2048 to 28672 x 8192 with 1 .. 4096 rows, 17
        // mixtures of 4 .. 128 experts with 4 .. 16384 rows, even and uneven, each with and without SiLU-gate), those of the kernels near
        // the fastest with more weight: 19 .. 26 % (rms) from each.  What they choose takes 1.02 times as long as the best of the kernels on
        // average (matrices and mixtures that the fit has not seen: 1.03 and 1.04), more than 1.15 times at 41 of the 1313 products --
        // among them 16 rows by 28672 x 8192 with SiLU-gate, 32.9 us on TILE_32x128, 26.9 on TILE_16x64 -- and at most 1.36 times (128 rows
        // in 8 uneven groups by 4096 x 14336).  How uneven the groups are the rule cannot know: 4096 rows in 60 by 2050 x 1376 take 46.4 us
        // on TILE_128x128 and 54.1 on TILE_64x128 if they are of one size, 54.0 and 49.7 if not.
        struct KernelFacts
        {
            int rows, cols, ranges, per_cu, step_values;
            bool gate;
            float start, turn, step, wait, off, rate;
        };
        constexpr KernelFacts FACTS[KERNELS] = {
            // (behind each: a product at which it is the fastest and is chosen, its time and that of the next)
            {16, 16, 8, 3, 128, false, 2.88f, 0.11f, 0.417f, 0.392f, 0.00f, 4.98f},  // ROWS_16x16: 2 rows by 4096 x 11008 in 7.9 us, the next best 9.8
            {16, 32, 4, 5, 128, true, 2.62f, 0.02f, 0.311f, 0.412f, 0.00f, 6.25f},   // ROWS_16x32: 24 rows by 2050 x 2080, SiLU-gate: 4.4 us, 6.5
            {8, 32, 2, 3, 256, true, 3.85f, 1.50f, 0.211f, 0.306f, 0.33f, 10.90f},   // TILE_8x32: 4 rows, 8 experts of 11008 x 4096: 18.3 us, 18.9
            {16, 32, 1, 4, 256, true, 3.63f, 1.56f, 0.112f, 0.235f, 0.48f, 8.02f},   // TILE_16x32: 16 rows by 22016 x 4096, SiLU-gate: 11.4 us, 13.0
            {16, 32, 2, 2, 256, true, 4.00f, 1.27f, 0.250f, 0.233f, 0.38f, 8.19f},   // TILE_16x32_2: 32 rows by 4096 x 11008, SiLU-gate: 10.7 us, 12.1
            {16, 32, 4, 1, 256, true, 3.32f, 1.61f, 0.515f, 0.515f, 0.59f, 6.34f},   // TILE_16x32_4: 96 rows by 1024 x 8192, SiLU-gate: 6.7 us, 7.4
            {16, 64, 2, 2, 256, true, 3.88f, 1.64f, 0.373f, 0.310f, 0.56f, 7.61f},   // TILE_16x64: 32 rows by 8192 x 8192, SiLU-gate: 13.5 us, 14.5
            {32, 64, 4, 1, 256, true, 3.32f, 1.74f, 0.920f, 0.920f, 0.46f, 5.67f},   // TILE_32x64: 384 rows by 1024 x 8192: 8.8 us, 11.1
            {32, 128, 1, 2, 256, true, 3.07f, 1.87f, 0.436f, 0.505f, 0.33f, 9.41f},  // TILE_32x128: 700 rows, 32 experts of 4096 x 1376, SiLU-gate: 28.7 us, 34.1
            {64, 64, 1, 2, 256, true, 4.05f, 1.56f, 0.293f, 0.276f, 0.27f, 6.53f},   // TILE_64x64: 1024 rows by 1000 x 5504, SiLU-gate: 11.5 us, 13.3
            {64, 128, 1, 2, 256, true, 3.46f, 2.83f, 0.533f, 0.688f, 0.27f, 5.26f},  // TILE_64x128: 700 rows, 16 uneven experts of 2880 x 2880: 26.7 us, 27.9
            {64, 128, 1, 1, 256, true, 4.17f, 3.21f, 0.474f, 0.474f, 0.32f, 6.24f},  // TILE_64x128_DEEP: 128 rows by 12288 x 4096: 13.3 us, 15.0
            {128, 128, 1, 2, 256, true, 4.41f, 4.14f, 0.636f, 0.871f, 0.23f, 6.12f}, // TILE_128x128: 4096 rows, 60 experts of 2050 x 1376, SiLU-gate: 40.1 us, 50.4
            {128, 128, 1, 1, 256, true, 5.12f, 4.25f, 0.662f, 0.662f, 0.23f, 6.64f}, // TILE_128x128_DEEP: 1024 rows by 4096 x 11008: 35.5 us, 47.1
            {256, 256, 1, 1, 256, true, 6.26f, 9.54f, 1.575f, 1.575f, 0.22f, 5.15f}, // TILE_256x256: 4096 rows by 12288 x 4096: 106 us, 145
        };

        // bytes of weights (every group's), activations and results
        inline float bytes_of(int M, int N, int K, bool gate, int experts)
        {
            const float matrices = (float)(experts > 0 ? experts < M ? experts : M : 1);
            return (matrices * N * (gate ? 2 : 1) + M) * K * (17 / 32.f) + (float)M * N * 2;
        }
        // estimated time; experts == 0: one product, else M rows in that many groups, whose sizes are not known here
        inline float estimate(const KernelFacts& k, int M, int N, int K, bool gate, int experts, int num_cu, float bytes)
        {
            // blocks of rows: a group ends in a block that is half full on average, and groups are of about one size
            float blocks = (float)((M + k.rows - 1) / k.rows);
            if (experts > 0)
            {
                const int groups = experts < M ? experts : M;
                blocks = groups * ((float)M / groups / k.rows + 0.5f);
                if (blocks < groups)
                    blocks = (float)groups;
            }
            const int all_steps = (K + k.step_values - 1) / k.step_values;
            int steps = (all_steps + k.ranges - 1) / k.ranges;
            if (k.step_values == 256 && k.ranges > 1)
            {
                steps = (steps + 1) & ~1;
                if (steps > all_steps)
                    steps = all_steps;
            }
            const float most = (float)(int)(blocks * column_tiles(N, k.cols, gate) / num_cu + 0.99999f); // workgroups of a CU
            const float rounds = (float)(((int)most + k.per_cu - 1) / k.per_cu);
            const float work = most * steps * k.step, wait = rounds * steps * k.wait, stream = bytes * 1e-6f / k.rate;
            const float steady = (work > wait ? work : wait) * (K % 256 ? 1 + k.off : 1);
            return k.start + k.turn * (rounds - 1) + (steady > stream ? steady : stream);
        }

        // whether a kernel has this form, in a grid that there can be
        constexpr bool fits(const KernelFacts& k, int M, int N, bool gate, int experts)
        {
            return (!gate || k.gate) && most_row_blocks(M, experts, k.rows) * column_tiles(N, k.cols, gate) <= MAX_WORKGROUPS;
        }

        // whether the library has a kernel for a product (experts == 0: one weight matrix): it takes these sizes, and some kernel's grid holds
        // their tiles
        constexpr bool servable(int M, int N, int K, bool gate, int experts)
        {
            if (!product_supported(M, N, K, gate, experts))
                return false;
            for (int k = 0; k < KERNELS; ++k)
                if (fits(FACTS[k], M, N, gate, experts))
                    return true;
            return false;
        }

        // the kernel with the lowest estimate of those that fit; KERNELS: none does
        inline Kernel choose(int M, int N, int K, bool gate, int experts, int num_cu)
        {
            const float bytes = bytes_of(M, N, K, gate, experts);
            int best = KERNELS;
            float time = 0;
            // (unrolled: divisions by constants, 0.13 us in place of 0.38)
#pragma GCC unroll 16
            for (int k = 0; k < KERNELS; ++k)
            {
                if (!fits(FACTS[k], M, N, gate, experts))
                    continue;
                const float t = estimate(FACTS[k], M, N, K, gate, experts, num_cu, bytes);
                if (best == KERNELS || t < time)
                    best = k, time = t;
            }
            return (Kernel)best;
        }
    } // namespace mx
} // namespace nnf
