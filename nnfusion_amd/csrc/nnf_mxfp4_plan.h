// Which kernel serves an MXFP4 product and what it needs: shared by the library and the emitters (host arithmetic only).
#pragma once

#include <stddef.h>

namespace nnf
{
    namespace mx
    {
        constexpr int MAX_K = 1 << 22; // byte offsets inside a tile of 256 rows stay below 2^31
        constexpr int scale_bytes(int K) { return ((K >> 5) + 15) & ~15; }
        constexpr bool supported(int K) { return K > 0 && K % 32 == 0 && K <= MAX_K; }

        struct Plan
        {
            bool tiles;     // the kernel through LDS (else: the one for a few rows)
            int row_shift;  // log2 of the rows of a block
            int row_blocks; // that there are at most
        };

        inline Plan plan(int experts, int M, int N, int K, bool gate, bool grouped)
        {
            (void)N, (void)K, (void)gate;
            const long long mean = grouped ? ((long long)M + experts - 1) / experts : M;
            Plan p = {};
            p.tiles = mean > 64;
            p.row_shift = p.tiles ? (mean > 1024 ? 8 : mean > 64 ? 7 : 6) : mean > 32 ? 6 : mean > 16 ? 5 : 4;
            // every group may end in a block of its own, which has a row at least
            const long long rows = 1LL << p.row_shift;
            const long long blocks = grouped ? (M + (long long)(experts < M ? experts : M) * (rows - 1)) / rows : (M + rows - 1) / rows;
            p.row_blocks = (int)blocks;
            return p;
        }
    } // namespace mx
} // namespace nnf
