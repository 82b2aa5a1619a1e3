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
        // quantising takes units of 512 values of a row, up to four to a workgroup, or blocks of 128 x 128; a grid has fewer than 2^32 threads
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
            TILE_128x128,
            TILE_256x256,
            KERNELS
        };
        struct KernelFacts
        {
            int rows, cols, ranges;
        };
        constexpr KernelFacts FACTS[KERNELS] = {{16, 32, 1}, {16, 32, 2}, {16, 32, 4}, {32, 64, 4}, {64, 64, 1}, {64, 128, 1}, {128, 128, 1}, {256, 256, 1}};

        constexpr bool fits(const KernelFacts& k, int M, int N, bool gate, int experts)
        {
            return most_row_blocks(M, experts, k.rows) * column_tiles(N, k.cols, gate) <= MAX_WORKGROUPS;
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
        inline Kernel choose(int M, int N, int K, bool gate, int experts, int num_cu)
        {
            const int rows = experts > 0 ? M / (experts < M ? experts : M) : M;
            int k = rows <= 32 ? TILE_16x32_2 : rows <= 128 ? TILE_64x64 : rows < 1024 ? TILE_128x128 : TILE_256x256;
            while (k < KERNELS - 1 && !fits(FACTS[k], M, N, gate, experts))
                ++k;
            return (Kernel)k;
        }
    } // namespace fp8
} // namespace nnf
