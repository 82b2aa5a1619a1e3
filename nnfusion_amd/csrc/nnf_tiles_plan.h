// How products over tiles of rows, grouped by expert or not, are counted: shared by the library and the emitters (host arithmetic only).
#pragma once

namespace nnf
{
    // blocks of `rows` rows that there are at most, of M rows in `experts` groups (0: one product): every group may end in a block of its
    // own, which has a row at least
    constexpr long long most_row_blocks(int M, int experts, int rows)
    {
        const long long groups = experts == 0 ? 1 : experts < M ? experts : M;
        return (M + groups * (rows - 1)) / rows;
    }
    // tiles of columns of Y, `cols` weight rows each
    constexpr int column_tiles(int N, int cols, bool gate) { return (int)(((long long)N + (gate ? cols / 2 : cols) - 1) / (gate ? cols / 2 : cols)); }
} // namespace nnf
