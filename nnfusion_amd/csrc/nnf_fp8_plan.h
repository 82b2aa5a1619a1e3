// Which kernel serves a product in block-scaled 8-bit floating point: shared by the library and the emitters (host arithmetic only).
#pragma once

#include "nnf_tiles_plan.h"

#include <stddef.h>

namespace nnf
{
    namespace fp8
    {
        constexpr int BLOCK = 128; // values along K, and rows of weights, of a scale
        constexpr int blocks_of(int size) { return size / BLOCK + (size % BLOCK != 0); }

        constexpr int MAX_K = 1 << 22; // byte offsets inside a tile of 256 rows stay below 2^31
        // rows of codes start on 16 bytes
        constexpr bool supported(int K) { return K > 0 && K % 16 == 0 && K <= MAX_K; }
        // quantising takes units of 512 values of a row or more, or blocks of 128 x 128; a grid has fewer than 2^32 threads
        constexpr int row_units(int K) { return (K + 511) / 512; }
        constexpr bool convertible(int rows, int K) { return supported(K) && (long long)rows * row_units(K) <= 1 << 24; }
        constexpr long long MAX_WORKGROUPS = (1 << 23) - 1; // a grid has fewer than 2^32 threads, and none of these kernels more than 512 in a workgroup
        constexpr bool weights_convertible(int matrices, int N, int K)
        {
            return supported(K) && (long long)blocks_of(N) * blocks_of(K) <= MAX_WORKGROUPS / matrices;
        }

        // sizes that a product may have (experts == 0: one weight matrix).  With SiLU-gate the bytes from a gate row to its up row are counted
        // in 32 bits; groups are looked through 64 at a time, and the first number behind them is an int too
        constexpr bool product_supported(int M, int N, int K, bool gate, int experts)
        {
            return supported(K) && M <= 1 << 30 && N <= 1 << 29 && (!gate || (long long)N * K < 1LL << 31) && experts <= 1 << 30;
        }

        // activation rows x weight rows of a workgroup's tile
        enum Kernel
        {
            TILE_16x32, // a wavefront for each range of K: one
            TILE_16x32_2, // two
            TILE_16x32_4, // four
            TILE_32x64, // four
            TILE_64x64, // the wavefronts share the tile and all of K
            TILE_64x128,
            TILE_128x256,
            TILE_256x256,
            ROWS_16x16, // operands straight into registers, a wavefront for each range of K: four; with SiLU-gate 16 gate rows and 16 up rows
            ROWS_16x32, // four; with SiLU-gate 32 and 32
            KERNELS
        };
        // What is known of a kernel: its tile, ranges of K, workgroups that a CU holds at once, and the constants of its time in us,
        //   start + turn * (rounds - 1) + max(step * workgroups of a CU * steps * (1 + off), wait * rounds * steps * (1 + off), bytes / rate)
        // with steps of 128 values, the rounds of workgroups that a CU runs and `off` where rows do not start on lines of memory (K no multiple of
        // 128); a step of the kernels without LDS goes by the lines that it loads, of weights and of the activation rows there are.  They are chosen for
        // the choice that comes of them, not for the times (which they give within 12 .. 20 %), by 1194 products, each on every kernel with its weights
        // from HBM: 15 matrices from 512 x 2048 to 28672 x 8192 with 1 .. 4096 rows, 13 mixtures of 4 .. 256 experts with 4 .. 16000 rows, even and uneven,
        // each with and without SiLU-gate.  Timed anew on other cards (profiles/fp8_product_timings.csv, by which a test holds the choice), what they choose
        // takes 1.010 times as long as the best kernel on average, 1.004 with one matrix and 1.015 with many; 1.009 with 64 .. 2000 rows, and above.  More than
        // 1.15 times at 9, at most 1.26 times (8192 rows in 60 even groups by 2 x 2050 x 1376, SiLU-gate: 186 us on TILE_128x256, 148 on
        // TILE_256x256).  Without any one of the kernels the best of the others would take 1.001 .. 1.019 times as long on average, 1.09 .. 1.43 times at worst.
        struct KernelFacts
        {
            int rows, cols, gate_cols, ranges, per_cu; // (gate_cols: with SiLU-gate, where that differs: the kernels without LDS)
            float start, turn, step, wait, off, rate;
        };
        constexpr int tiles_of_columns(const KernelFacts& k, int N, bool gate) { return column_tiles(N, gate ? k.gate_cols : k.cols, gate); }
        constexpr KernelFacts FACTS[KERNELS] = {
            {16, 32, 32, 1, 6, 3.970f, 0.797f, 0.123f, 0.288f, 0.055f, 6.590f},
            {16, 32, 32, 2, 3, 3.356f, 0.984f, 0.209f, 0.276f, 0.535f, 6.682f},
            {16, 32, 32, 4, 1, 4.590f, 3.822f, 0.254f, 0.294f, 0.504f, 8.090f},
            {32, 64, 64, 4, 1, 3.345f, 2.858f, 0.033f, 0.836f, 0.409f, 4.530f},
            {64, 64, 64, 1, 2, 4.164f, 1.052f, 0.288f, 0.274f, 0.284f, 6.613f},
            {64, 128, 128, 1, 2, 4.436f, 0.618f, 0.426f, 0.020f, 0.342f, 6.409f},
            {128, 256, 256, 1, 1, 4.128f, 3.464f, 0.945f, 0.945f, 0.259f, 6.195f},
            {256, 256, 256, 1, 1, 2.958f, 5.072f, 0.020f, 1.475f, 0.150f, 4.430f},
            {16, 16, 32, 4, 4, 2.699f, 0.679f, 0.420f, 0.466f, 0.020f, 6.586f},
            {16, 32, 64, 4, 4, 2.388f, 0.410f, 0.441f, 0.529f, 0.019f, 6.016f},
        };

        // bytes of weights (every group's), activations and results
        inline float bytes_of(int M, int N, int K, bool gate, int experts)
        {
            const float matrices = (float)(experts > 0 ? experts < M ? experts : M : 1);
            return (matrices * N * (gate ? 2 : 1) + M) * K + (float)M * N * 2;
        }
        // estimated time; experts == 0: one product, else M rows in that many groups, whose sizes are not known here
        inline float estimate(const KernelFacts& k, int M, int N, int K, bool gate, int experts, int num_cu, float bytes)
        {
            // blocks of rows: a group ends in a block that is half full on average, and groups are of about one size
            float blocks = (float)((M + k.rows - 1) / k.rows), of_group = (float)M;
            if (experts > 0)
            {
                const int groups = experts < M ? experts : M;
                of_group = (float)M / groups;
                blocks = groups * (of_group / k.rows + 0.5f);
                if (blocks < groups)
                    blocks = (float)groups;
            }
            float lines = 1;
            if (k.gate_cols != k.cols)
                lines = ((gate ? k.gate_cols : k.cols) + (of_group < k.rows ? of_group : k.rows)) * (1 / 32.f);
            const int steps = (blocks_of(K) + k.ranges - 1) / k.ranges;
            const float most = (float)(int)(blocks * tiles_of_columns(k, N, gate) / num_cu + 0.99999f); // workgroups of a CU
            const float rounds = (float)(((int)most + k.per_cu - 1) / k.per_cu);
            const float work = most * steps * k.step * lines, wait = rounds * steps * k.wait * lines, stream = bytes * 1e-6f / k.rate;
            const float steady = (work > wait ? work : wait) * (K % BLOCK ? 1 + k.off : 1);
            return k.start + k.turn * (rounds - 1) + (steady > stream ? steady : stream);
        }

        constexpr bool fits(const KernelFacts& k, int M, int N, bool gate, int experts)
        {
            return most_row_blocks(M, experts, k.rows) * tiles_of_columns(k, N, gate) <= MAX_WORKGROUPS;
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
            // (unrolled: divisions by constants)
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
    } // namespace fp8
} // namespace nnf
