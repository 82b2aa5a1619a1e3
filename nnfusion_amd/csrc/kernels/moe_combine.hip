// The experts' rows back to their tokens: y[t] = residual[t] + sum_j weights[t, j] x[positions[t, j]], fp32 sums in the order of j, rounded once.
//
// One pass over memory, bound by HBM: a wavefront has 512 columns of a token, eight to a lane, and asks for up to eight experts' pieces
// ahead of the first sum.  Experts' rows that would not stay in the 256 MB cache at the memory are read past the caches: 8 rows each of 8192 tokens, 4096
// columns, onto a residual in 106 .. 114 us, 132 without (5.9 .. 6.3 TB/s; a copy of 1 GiB runs at 5.0 .. 5.2, a read at up to 7.0); at 128 MB of rows it would be 30.0 in place of 29.2.
#include "moe_launch.h"
#include "nnf_device.h"

namespace nnf
{
    namespace
    {
        typedef __bf16 bf16_t;
        constexpr int WAVES = 4, COLUMNS = 8 * WAVE, AT_ONCE = 8;
        static_assert(moe::combine_units(COLUMNS) == 1 && moe::combine_units(COLUMNS + 1) == 2, "units of a wavefront");

        // bytes of experts' rows from which on they are read past the caches
        constexpr long long PASSING = 256ll << 20;

        // WIDE: all rows start on 16 bytes.  PASS: x is read past the caches.  y may be the residual: a lane reads what it writes, ahead of that
        template <class T, bool WIDE, bool PASS>
        __global__ __launch_bounds__(WAVES* WAVE) void moe_combine_kernel(const T* __restrict__ x, const float* __restrict__ weights,
                                                                         const int* __restrict__ positions, const T* residual, T* y,
                                                                         int units, int row_units, int rows, int k, int N)
        {
            typedef T Eight __attribute__((ext_vector_type(8)));
            const int unit = (int)blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
            if (unit >= units)
                return;
            const int t = unit / row_units, n = (unit - t * row_units) * COLUMNS + (threadIdx.x & (WAVE - 1)) * 8;
            if (n >= N)
                return;
            const int last = min(N - n, 8);
            const auto piece = [&](const T* row, auto pass) {
                Eight v;
                if constexpr (WIDE && pass)
                    v = __builtin_bit_cast(Eight, __builtin_nontemporal_load(reinterpret_cast<const uintx4*>(row + n)));
                else if constexpr (WIDE)
                    v = *reinterpret_cast<const Eight*>(row + n);
                else
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        v[i] = i < last ? row[n + i] : (T)0.0f;
                return v;
            };
            float sum[8] = {};
            for (int j0 = 0; j0 < k; j0 += AT_ONCE)
            {
                Eight v[AT_ONCE];
                float w[AT_ONCE];
#pragma unroll
                for (int j = 0; j < AT_ONCE; ++j)
                {
                    w[j] = 0;
                    if (j0 + j < k)
                    {
                        const int at = positions[(size_t)t * k + j0 + j];
                        w[j] = weights[(size_t)t * k + j0 + j];
                        if (at < 0 || at >= rows)
                            w[j] = 0;
                        if (w[j] != 0)
                            v[j] = piece(x + (size_t)at * N, std::bool_constant<PASS>{});
                    }
                }
#pragma unroll
                for (int j = 0; j < AT_ONCE; ++j)
                    if (w[j] != 0) // (a weight of zero takes nothing from its row, whatever lies there)
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            sum[i] = __builtin_fmaf(w[j], (float)v[j][i], sum[i]);
            }
            if (residual)
            {
                const Eight v = piece(residual + (size_t)t * N, std::false_type{});
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    sum[i] += (float)v[i];
            }
            T* const to = y + (size_t)t * N + n;
            if constexpr (WIDE)
            {
                Eight v;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    v[i] = (T)sum[i];
                *reinterpret_cast<Eight*>(to) = v;
            }
            else
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < last)
                        to[i] = (T)sum[i];
        }

        template <class T>
        hipError_t launch(hipStream_t s, const void* x, const float* weights, const int* positions, const void* residual, void* y, int tokens, int rows, int k, int N)
        {
            const int row_units = moe::combine_units(N), units = tokens * row_units, groups = (units + WAVES - 1) / WAVES;
            const bool wide = N % 8 == 0 && ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(y)) & 15) == 0;
            const bool pass = (long long)tokens * k * N * 2 >= PASSING;
            const auto kernel = !wide ? moe_combine_kernel<T, false, false> : pass ? moe_combine_kernel<T, true, true> : moe_combine_kernel<T, true, false>;
            kernel<<<groups, WAVES * WAVE, 0, s>>>((const T*)x, weights, positions, (const T*)residual, (T*)y, units, row_units, rows, k, N);
            return hipGetLastError();
        }
    } // namespace

    hipError_t launch_moe_combine(hipStream_t s, const void* x, const float* weights, const int* positions, const void* residual, void* y, int tokens, int rows, int k,
                                  int N, bool bf16)
    {
        return bf16 ? launch<bf16_t>(s, x, weights, positions, residual, y, tokens, rows, k, N)
                    : launch<half_t>(s, x, weights, positions, residual, y, tokens, rows, k, N);
    }
} // namespace nnf
