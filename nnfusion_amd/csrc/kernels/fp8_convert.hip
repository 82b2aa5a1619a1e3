// fp16 or bf16 -> block-scaled E4M3 (fp8.h): rows, picked by an index or not, with a scale for each 128 values, and weight matrices with
// a scale for each block of 128 x 128.
//
// scale = max(largest magnitude, 2^-64) / 448, code = E4M3(x / scale): both quotients rounded to fp32 as IEEE has it, so that a code next to a tie
// is the one that any fp32 implementation gets.  x / scale is the product with the scale's rounded inverse, put right twice by its remainder
// (each step an fma: the first leaves less than half a step and a bit, the second rounds correctly); the bound of 2^-64 keeps all of that
// away from subnormals.  A block with an infinity or NaN: scale NaN, codes 0.
//
// One pass over memory, two bytes read and one written a value.
#include "fp8_launch.h"
#include "nnf_launch.h"

namespace nnf
{
    namespace
    {
        using namespace fp8;

        constexpr int CONVERT_THREADS = 256;
        constexpr int WAVES = CONVERT_THREADS / WAVE;

        __device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b)
        {
            typedef unsigned short ushortx2 __attribute__((ext_vector_type(2)));
            return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushortx2, a), __builtin_bit_cast(ushortx2, b)));
        }
        // the largest magnitude of eight values, in either half, as the bit pattern of their type: these are ordered like the numbers
        __device__ __forceinline__ uint32_t top_of(uintx4 v)
        {
            return max_u16x2(max_u16x2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu), max_u16x2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
        }
        __device__ __forceinline__ uint32_t top_of_16_lanes(uint32_t top)
        {
            top = max_u16x2(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x128, 0xF, 0xF, false)); // row_ror:8
            top = max_u16x2(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x124, 0xF, 0xF, false)); // row_ror:4
            top = max_u16x2(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x122, 0xF, 0xF, false)); // row_ror:2
            top = max_u16x2(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x121, 0xF, 0xF, false)); // row_ror:1
            return max(top >> 16, top & 0xFFFFu);
        }
        template <bool BF16>
        __device__ __forceinline__ float number(uint32_t bits)
        {
            return BF16 ? __builtin_bit_cast(float, bits << 16) : (float)__builtin_bit_cast(half_t, (uint16_t)bits);
        }
        template <bool BF16>
        __device__ __forceinline__ float scale_of(uint32_t top)
        {
            return top < (BF16 ? 0x7F80u : 0x7C00u) ? fmaxf(number<BF16>(top), 0x1p-64f) / 448.0f : __builtin_nanf("");
        }
        // eight values' codes
        template <bool BF16>
        __device__ __forceinline__ uintx2 codes_of(uintx4 v, float scale)
        {
            const float inverse = 1.0f / scale;
            const bool fine = scale == scale;
            float q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
            {
                const float x = number<BF16>(v[i / 2] >> (i % 2 * 16) & 0xFFFFu);
                float y = x * inverse;
                y = __builtin_fmaf(__builtin_fmaf(-y, scale, x), inverse, y);
                q[i] = __builtin_copysignf(__builtin_fmaf(__builtin_fmaf(-y, scale, x), inverse, y), x); // (of -0 the sums above are 0)
            }
            uintx2 c;
#pragma unroll
            for (int h = 0; h < 2; ++h)
            {
                int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h], q[4 * h + 1], 0, false);
                w = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h + 2], q[4 * h + 3], w, true);
                c[h] = fine ? (uint32_t)w : 0u;
            }
            return c;
        }

        // A wavefront takes UNITS units of 512 values of one row, eight to a lane, all their loads ahead of the first use
        template <int UNITS, bool BF16>
        __global__ __launch_bounds__(CONVERT_THREADS) void fp8_quantize_kernel(const uint16_t* __restrict__ x, const int* __restrict__ index, uint8_t* __restrict__ codes,
                                                                               float* __restrict__ scales, int units, int row_units, int rows, int source_rows, int K)
        {
            const int lane = threadIdx.x & (WAVE - 1);
            const int first = ((int)blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE)) * UNITS;
            int row[UNITS], unit[UNITS];
            row[0] = first / row_units;
            unit[0] = first - row[0] * row_units;
#pragma unroll
            for (int i = 1; i < UNITS; ++i)
            {
                const bool next = unit[i - 1] + 1 == row_units;
                row[i] = row[i - 1] + (next ? 1 : 0);
                unit[i] = next ? 0 : unit[i - 1] + 1;
            }
            uintx4 v[UNITS];
#pragma unroll
            for (int i = 0; i < UNITS; ++i)
            {
                const int k = unit[i] * 512 + lane * 8;
                v[i] = uintx4{0, 0, 0, 0};
                if (first + i < units && k < K)
                {
                    const long long from = index ? index[row[i]] : (long long)row[i];
                    if (from >= 0 && from < source_rows)
                        v[i] = *reinterpret_cast<const uintx4*>(x + from * K + k);
                }
            }
#pragma unroll
            for (int i = 0; i < UNITS; ++i)
            {
                if (first + i >= units)
                    return;
                const float scale = scale_of<BF16>(top_of_16_lanes(top_of(v[i])));
                const uintx2 c = codes_of<BF16>(v[i], scale);
                const int k = unit[i] * 512 + lane * 8;
                if (k < K)
                {
                    *reinterpret_cast<uintx2*>(codes + (size_t)row[i] * K + k) = c;
                    if ((lane & 15) == 0)
                        scales[(size_t)(k >> 7) * rows + row[i]] = scale;
                }
            }
        }

        // A workgroup has a block of 128 x 128, a wavefront 32 rows of it, four rows to a load
        template <bool BF16>
        __global__ __launch_bounds__(CONVERT_THREADS) void fp8_quantize_weights_kernel(const uint16_t* __restrict__ w, uint8_t* __restrict__ codes,
                                                                                       float* __restrict__ scales, int row_blocks, int N, int K)
        {
            __shared__ uint32_t tops[WAVES];
            const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE, blocks = blocks_of(K);
            const int block = (int)blockIdx.x / blocks, kb = (int)blockIdx.x - block * blocks; // block of rows, of all matrices'
            const int matrix = block / row_blocks;
            const int n0 = (block - matrix * row_blocks) * BLOCK + wave * 32 + (lane >> 4), k = kb * BLOCK + (lane & 15) * 8;
            const size_t base = (size_t)matrix * N;
            constexpr int LOADS = 8;
            uintx4 v[LOADS];
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
            {
                v[i] = uintx4{0, 0, 0, 0};
                if (n0 + i * 4 < N && k < K)
                    v[i] = *reinterpret_cast<const uintx4*>(w + (base + n0 + i * 4) * K + k);
            }
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                top = max_u16x2(top, top_of(v[i]));
            top = top_of_16_lanes(top);
            top = max(top, (uint32_t)__shfl_xor((int)top, 16));
            top = max(top, (uint32_t)__shfl_xor((int)top, 32));
            if (lane == 0)
                tops[wave] = top;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < WAVES; ++i)
                top = max(top, tops[i]);
            const float scale = scale_of<BF16>(top);
            if (threadIdx.x == 0)
                scales[blockIdx.x] = scale;
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                if (n0 + i * 4 < N && k < K)
                    *reinterpret_cast<uintx2*>(codes + (base + n0 + i * 4) * K + k) = codes_of<BF16>(v[i], scale);
        }

        template <bool BF16>
        hipError_t launch_rows(hipStream_t s, const void* x, const void* index, void* codes, float* scales, int rows, int source_rows, int K)
        {
            // four units a wavefront once these fill the CUs; one below, where the time is one load's latency
            constexpr int MANY = 4;
            const int each = row_units(K), units = rows * each;
            if (units < 256 * WAVES * MANY * 2)
                fp8_quantize_kernel<1, BF16><<<(units + WAVES - 1) / WAVES, CONVERT_THREADS, 0, s>>>((const uint16_t*)x, (const int*)index, (uint8_t*)codes, scales, units,
                                                                                                      each, rows, source_rows, K);
            else
                fp8_quantize_kernel<MANY, BF16><<<(units + WAVES * MANY - 1) / (WAVES * MANY), CONVERT_THREADS, 0, s>>>(
                    (const uint16_t*)x, (const int*)index, (uint8_t*)codes, scales, units, each, rows, source_rows, K);
            return hipGetLastError();
        }
        template <bool BF16>
        hipError_t launch_weights(hipStream_t s, const void* w, void* codes, float* scales, int matrices, int N, int K)
        {
            fp8_quantize_weights_kernel<BF16><<<matrices * blocks_of(N) * blocks_of(K), CONVERT_THREADS, 0, s>>>((const uint16_t*)w, (uint8_t*)codes, scales, blocks_of(N), N, K);
            return hipGetLastError();
        }
    } // namespace

    hipError_t launch_fp8_quantize(hipStream_t s, const void* x, bool bf16, const void* index, void* codes, float* scales, int rows, int source_rows, int K)
    {
        return bf16 ? launch_rows<true>(s, x, index, codes, scales, rows, source_rows, K) : launch_rows<false>(s, x, index, codes, scales, rows, source_rows, K);
    }

    hipError_t launch_fp8_quantize_weights(hipStream_t s, const void* w, bool bf16, void* codes, float* scales, int matrices, int N, int K)
    {
        return bf16 ? launch_weights<true>(s, w, codes, scales, matrices, N, K) : launch_weights<false>(s, w, codes, scales, matrices, N, K);
    }
} // namespace nnf
