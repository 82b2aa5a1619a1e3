// fp16 <-> MXFP4 (mxfp4.h): quantising rows, picked by an index or not, and reading them back.
//
// Both are one pass over memory: 2 bytes of fp16 and 17/32 byte of MXFP4 per value.  A wavefront takes units of 512 values of one row, eight
// to a lane: 16 bytes of fp16, 4 bytes of codes, a block of 32 values to each four lanes, its scale byte by way of the lanes'
// maximum.  A unit is 1 KiB, 256 bytes and 16 bytes in memory order; the row of scale bytes is padded to 16, so units never share one.
// The hardware's conversion does the division by the power of two, the rounding and the saturation of a pair of values at once.
//
// Bound by HBM from some thousand units on: 22016 x 4096 quantised in 41 us and read back in 43 where each runs over buffers beyond the
// cache, one launch after the other (5.6 and 5.3 TB/s; a copy of 1 GiB runs at 5.2); 4000 x 5504 in 12.0 and 13.1.  In turn, the results
// of one read by the other, the two take 89 us together; a trace then shows 54 and 34, as what the 256 MB cache holds of a
// kernel's results goes out under the next one.  Below, by the launch: 256 x 11008 in 3.0 us, 16 x 4096 in 2.1 (launches in a graph; 1.2
// and 1.4 us of kernel for one row).
#include "mxfp4.h"
#include "nnf_launch.h"

namespace nnf
{
    namespace
    {
        using namespace mx;

        constexpr int CONVERT_THREADS = 256;
        constexpr int WAVES = CONVERT_THREADS / WAVE;

        // the larger of two pairs of 16-bit magnitudes
        __device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b)
        {
            typedef unsigned short ushortx2 __attribute__((ext_vector_type(2)));
            return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushortx2, a), __builtin_bit_cast(ushortx2, b)));
        }

        // where the units of a wavefront lie: UNITS of them from its first on, their rows and places in them found with one division
        template <int UNITS>
        struct Place
        {
            int first; // unit of the first
            int row[UNITS];
            int unit[UNITS];
            __device__ __forceinline__ Place(int row_units)
            {
                first = ((int)blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE)) * UNITS;
                row[0] = first / row_units;
                unit[0] = first - row[0] * row_units;
#pragma unroll
                for (int i = 1; i < UNITS; ++i)
                {
                    const bool next = unit[i - 1] + 1 == row_units;
                    row[i] = row[i - 1] + (next ? 1 : 0);
                    unit[i] = next ? 0 : unit[i - 1] + 1;
                }
            }
        };

        template <int UNITS>
        __global__ __launch_bounds__(CONVERT_THREADS) void mxfp4_quantize_kernel(const half_t* __restrict__ x, const int* __restrict__ index,
                                                                                 uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                                                 int units, int row_units, int source_rows, int K)
        {
            const int lane = threadIdx.x & (WAVE - 1);
            const Place<UNITS> at(row_units);
            uintx4 v[UNITS];
#pragma unroll
            for (int i = 0; i < UNITS; ++i)
            {
                const int k = at.unit[i] * 512 + lane * 8;
                v[i] = uintx4{0, 0, 0, 0};
                if (at.first + i < units && k < K)
                {
                    // (a row that is not there is a row of zeros)
                    const long long from = index ? index[at.row[i]] : (long long)at.row[i];
                    if (from >= 0 && from < source_rows)
                        v[i] = *reinterpret_cast<const uintx4*>(x + from * K + k);
                }
            }
#pragma unroll
            for (int i = 0; i < UNITS; ++i)
            {
                if (at.first + i >= units)
                    return;
                // the largest magnitude of the block as an fp16 bit pattern: these are ordered like the numbers, infinity and NaN above
                uint32_t top = max_u16x2(max_u16x2(v[i].x & 0x7FFF7FFFu, v[i].y & 0x7FFF7FFFu), max_u16x2(v[i].z & 0x7FFF7FFFu, v[i].w & 0x7FFF7FFFu));
                top = max_u16x2(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, false)); // 1,0,3,2
                top = max_u16x2(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, false)); // 2,3,0,1
                top = max(top >> 16, top & 0xFFFFu);
                // floor(log2(top)) - 2 + 127: the exponent field of the same number in fp32, where fp16's subnormals are normal
                const uint32_t exponent = __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(half_t, (uint16_t)top)) >> 23;
                const bool finite = top < 0x7C00u;
                const uint32_t byte = top == 0 ? 127u : finite ? exponent - 2 : 255u;
                const float scale = __builtin_bit_cast(float, byte << 23);
                uint32_t code = 0;
                // (the conversion divides by the scale's power of two, rounds to nearest even and saturates at 6)
                code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(code, as_half2(v[i].x), scale, 0);
                code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(code, as_half2(v[i].y), scale, 1);
                code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(code, as_half2(v[i].z), scale, 2);
                code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(code, as_half2(v[i].w), scale, 3);
                const int k = at.unit[i] * 512 + lane * 8;
                if (k < K)
                    *reinterpret_cast<uint32_t*>(codes + (size_t)at.row[i] * (K / 2) + k / 2) = finite ? code : 0u;
                if ((lane & 3) == 0)
                    scales[(size_t)(at.first + i) * 16 + lane / 4] = (uint8_t)byte; // (behind the row's end: 2^0)
            }
        }

        template <int UNITS>
        __global__ __launch_bounds__(CONVERT_THREADS) void mxfp4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                                                   half_t* __restrict__ y, int units, int row_units, int K)
        {
            const int lane = threadIdx.x & (WAVE - 1);
            const Place<UNITS> at(row_units);
            uint32_t code[UNITS], byte[UNITS];
#pragma unroll
            for (int i = 0; i < UNITS; ++i)
            {
                const int k = at.unit[i] * 512 + lane * 8;
                code[i] = 0, byte[i] = 127;
                if (at.first + i < units && k < K)
                {
                    code[i] = *reinterpret_cast<const uint32_t*>(codes + (size_t)at.row[i] * (K / 2) + k / 2);
                    byte[i] = scales[(size_t)(at.first + i) * 16 + lane / 4];
                }
            }
#pragma unroll
            for (int i = 0; i < UNITS; ++i)
            {
                const int k = at.unit[i] * 512 + lane * 8;
                if (at.first + i >= units || k >= K)
                    continue;
                // 6 * 2^-30 and 0.5 * 2^20 are beyond fp16 as any value outside these two is (a scale of 2^-127 has no normal fp32)
                const float scale = byte[i] == 255 ? __builtin_nanf("") : __builtin_bit_cast(float, min(max(byte[i], 127u - 30u), 127u + 20u) << 23);
                // the four-bit values exactly, then their products with the power of two, exact in fp32 and rounded once
                const half2_t h[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code[i], 1.0f, 0), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code[i], 1.0f, 1),
                                      __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code[i], 1.0f, 2), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code[i], 1.0f, 3)};
                half8_t out;
#pragma unroll
                for (int p = 0; p < 8; ++p)
                    out[p] = (half_t)((float)h[p / 2][p % 2] * scale);
                *reinterpret_cast<half8_t*>(y + (size_t)at.row[i] * K + k) = out;
            }
        }

        // f(units, units of a wavefront as a constant, units of a row, workgroups): four units a wavefront, all their loads ahead of the
        // first use, once these fill the CUs; one below, where the time is one load's latency and as many wavefronts as there are units
        // share it
        template <class F>
        hipError_t over_units(int rows, int K, F f)
        {
            constexpr int MANY = 4;
            const int units = rows * row_units(K);
            if (units < 256 * WAVES * MANY * 2)
                return f(units, std::integral_constant<int, 1>{}, row_units(K), (units + WAVES - 1) / WAVES);
            return f(units, std::integral_constant<int, MANY>{}, row_units(K), (units + WAVES * MANY - 1) / (WAVES * MANY));
        }
    } // namespace

    hipError_t launch_mxfp4_quantize(hipStream_t s, const void* x, const void* index, void* codes, void* scales, int rows, int source_rows, int K)
    {
        return over_units(rows, K, [&](int units, auto many, int row_units, int groups) {
            mxfp4_quantize_kernel<many><<<groups, CONVERT_THREADS, 0, s>>>((const half_t*)x, (const int*)index, (uint8_t*)codes,
                                                                                            (uint8_t*)scales, units, row_units, source_rows, K);
            return hipGetLastError();
        });
    }

    hipError_t launch_mxfp4_dequantize(hipStream_t s, const void* codes, const void* scales, void* y, int rows, int K)
    {
        return over_units(rows, K, [&](int units, auto many, int row_units, int groups) {
            mxfp4_dequantize_kernel<many><<<groups, CONVERT_THREADS, 0, s>>>((const uint8_t*)codes, (const uint8_t*)scales, (half_t*)y, units,
                                                                                              row_units, K);
            return hipGetLastError();
        });
    }
} // namespace nnf
