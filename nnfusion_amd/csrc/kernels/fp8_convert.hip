// fp16 or bf16 -> block-scaled E4M3 (fp8.h): rows, picked by an index or not, with a scale for each 128 values, and weight matrices with
// a scale for each block of 128 x 128.
//
// scale = max(largest magnitude, 2^-64) / 448, code = E4M3(x / scale): both quotients as IEEE rounds them to fp32, so that a code next to a tie is
// the one that any fp32 implementation gets.  Neither is divided for.  The scale is a product with the rounded 1 / 448 and one step of its
// remainder, exact for every significand of 11 bits.  x / scale is x (inverse + rest) rounded once, rest being what the rounded inverse of the scale lacks:
// off by 2^-41 before the rounding, where a quotient that is a tie of E4M3 but for the scale's rounding is never nearer than 2^-35 to a midpoint of
// fp32 and any other one is 2^-17 away from a tie.  Powers of two are kept out of it until the conversion, which takes them for nothing, so that no
// number leaves fp32's range.  A block with an infinity or NaN: scale NaN, codes 0.
//
// One pass over memory, two bytes read and one written a value: bound by HBM where there are enough of them -- 22016 x 4096 in 42 us as rows (6.4 TB/s; a copy
// of 1 GiB runs at 5.0 .. 5.2, a read at up to 7.0) and in 42 .. 44 as blocks of 128 x 128 (48 .. 50 where each call's results are new memory).  4000 of 1000
// rows of 5504 take 10.3 us, 4.8 of them bytes at a read's rate.  A lane takes 16
// values, so that a block's scale is made by eight lanes in place of 16, and a workgroup four rows at one place, whose scales lie side by side: with
// eight values and four places of one row 47, 12.2 us, and 17.4 in place of 10.8 for 32768 x 528; eight rows are as fast, 16 slower.  16 rows of
// 4096 in 2.1 us, of which a launch is 1.8.  Results go through the caches, as a product reads them next: past them, a product of 256 x 4096 x 4096
// behind takes 2 us longer.
#include "fp8_launch.h"
#include "nnf_launch.h"

namespace nnf
{
    namespace
    {
        using namespace fp8;

        constexpr int CONVERT_THREADS = 256;
        constexpr int WAVES = CONVERT_THREADS / WAVE;
        constexpr int ROWS = WAVES, ROWS_OF_GRID = 1 << 15; // rows of a workgroup; so many times that in y, the others in z

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
        // of eight lanes in the low half
        __device__ __forceinline__ uint32_t top_of_8_lanes(uint32_t top)
        {
            top = max_u16x2(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, false));  // quad_perm 1,0,3,2
            top = max_u16x2(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, false));  // 2,3,0,1
            top = max_u16x2(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x141, 0xF, 0xF, false)); // row_half_mirror
            return max(top >> 16, top & 0xFFFFu);
        }
        template <bool BF16>
        __device__ __forceinline__ float number(uint32_t bits)
        {
            return BF16 ? __builtin_bit_cast(float, bits << 16) : (float)__builtin_bit_cast(half_t, (uint16_t)bits);
        }
        // What a block's values are quantised with: x / scale = x (inverse + rest) / power, rest >= 0 (so that -0 stays what it is)
        struct Quotient
        {
            float scale, power, inverse, rest;
        };
        template <bool BF16>
        __device__ __forceinline__ Quotient quotient_of(uint32_t top)
        {
            constexpr float C = 1.0f / 448.0f;
            const float a = fmaxf(number<BF16>(top), 0x1p-64f), q = a * C;
            Quotient v;
            v.scale = __builtin_fmaf(__builtin_fmaf(-q, 448.0f, a), C, q);
            const uint32_t bits = __builtin_bit_cast(uint32_t, v.scale);
            const float m = __builtin_bit_cast(float, (bits & 0x007FFFFFu) | 0x3F800000u);
            v.power = __builtin_bit_cast(float, bits & 0x7F800000u);
            // (the hardware's inverse is good to a step: two steps lower it is below 1 / m)
            v.inverse = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, __builtin_amdgcn_rcpf(m)) - 2);
            v.rest = __builtin_fmaf(-m, v.inverse, 1.0f) * v.inverse;
            if (top >= (BF16 ? 0x7F80u : 0x7C00u))
                v.scale = __builtin_nanf("");
            return v;
        }
        // eight values' codes
        template <bool BF16>
        __device__ __forceinline__ uintx2 codes_of(uintx4 v, const Quotient& by)
        {
            typedef short shortx2 __attribute__((ext_vector_type(2)));
            float q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
            {
                const float x = BF16 ? __builtin_bit_cast(float, i & 1 ? v[i / 2] & 0xFFFF0000u : v[i / 2] << 16) : (float)as_half2(v[i / 2])[i & 1];
                q[i] = __builtin_fmaf(x, by.inverse, x * by.rest);
            }
            uintx2 c;
#pragma unroll
            for (int h = 0; h < 2; ++h)
            {
                shortx2 w = {};
                w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, q[4 * h], q[4 * h + 1], by.power, false);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, q[4 * h + 2], q[4 * h + 3], by.power, true);
                c[h] = by.scale == by.scale ? __builtin_bit_cast(uint32_t, w) : 0u;
            }
            return c;
        }

        // A wavefront takes 512 or 1024 values of a row, EACH = 8 or 16 to a lane; a workgroup the same of four rows
        template <bool BF16, int EACH>
        __global__ __launch_bounds__(CONVERT_THREADS) void fp8_quantize_kernel(const uint16_t* __restrict__ x, const int* __restrict__ index, uint8_t* __restrict__ codes,
                                                                               float* __restrict__ scales, int rows, int source_rows, int K)
        {
            constexpr int PIECES = EACH / 8;
            const int lane = threadIdx.x & (WAVE - 1), row = (int)(blockIdx.z * ROWS_OF_GRID + blockIdx.y) * ROWS + __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
            const int k = ((int)blockIdx.x * WAVE + lane) * EACH;
            if (row >= rows)
                return;
            const int from = index ? index[row] : row;
            uintx4 v[PIECES] = {}; // (a row that is not there is a row of zeros)
            if (k < K && from >= 0 && from < source_rows)
#pragma unroll
                for (int i = 0; i < PIECES; ++i)
                    v[i] = *reinterpret_cast<const uintx4*>(x + (size_t)from * K + k + i * 8);
            uint32_t top = top_of(v[0]);
            if constexpr (PIECES == 2)
                top = top_of_8_lanes(max_u16x2(top, top_of(v[1])));
            else
                top = top_of_16_lanes(top);
            const Quotient by = quotient_of<BF16>(top);
            uintx2 c[PIECES];
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
                c[i] = codes_of<BF16>(v[i], by);
            if (k < K)
            {
                uint8_t* const to = codes + (size_t)row * K + k;
                if constexpr (PIECES == 2)
                    *reinterpret_cast<uintx4*>(to) = uintx4{c[0].x, c[0].y, c[1].x, c[1].y};
                else
                    *reinterpret_cast<uintx2*>(to) = c[0];
                if (lane % (BLOCK / EACH) == 0)
                    scales[(size_t)(k >> 7) * rows + row] = by.scale;
            }
        }

        // A workgroup has a block of 128 x 128, a wavefront 16 rows of it, four rows to a load (32 rows each of four wavefronts: 52 us in place of 48 for
        // 22016 x 4096; 16 wavefronts 50)
        constexpr int BLOCK_WAVES = 8;
        template <bool BF16>
        __global__ __launch_bounds__(BLOCK_WAVES* WAVE) void fp8_quantize_weights_kernel(const uint16_t* __restrict__ w, uint8_t* __restrict__ codes,
                                                                                       float* __restrict__ scales, int row_blocks, int N, int K)
        {
            constexpr int LOADS = BLOCK / 4 / BLOCK_WAVES;
            __shared__ uint32_t tops[BLOCK_WAVES];
            const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE, blocks = blocks_of(K);
            const int block = (int)blockIdx.x / blocks, kb = (int)blockIdx.x - block * blocks; // block of rows, of all matrices'
            const int matrix = block / row_blocks;
            const int n0 = (block - matrix * row_blocks) * BLOCK + wave * (LOADS * 4) + (lane >> 4), k = kb * BLOCK + (lane & 15) * 8;
            const size_t base = (size_t)matrix * N;
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
            for (int i = 0; i < BLOCK_WAVES; ++i)
                top = max(top, tops[i]);
            const Quotient by = quotient_of<BF16>(top);
            if (threadIdx.x == 0)
                scales[blockIdx.x] = by.scale;
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                if (n0 + i * 4 < N && k < K)
                    *reinterpret_cast<uintx2*>(codes + (base + n0 + i * 4) * K + k) = codes_of<BF16>(v[i], by);
        }

        template <bool BF16, int EACH>
        hipError_t launch_rows(hipStream_t s, const void* x, const void* index, void* codes, float* scales, int rows, int source_rows, int K)
        {
            const int units = (K + WAVE * EACH - 1) / (WAVE * EACH), of_rows = (rows + ROWS - 1) / ROWS;
            const dim3 grid(units, of_rows < ROWS_OF_GRID ? of_rows : ROWS_OF_GRID, (of_rows + ROWS_OF_GRID - 1) / ROWS_OF_GRID);
            fp8_quantize_kernel<BF16, EACH><<<grid, CONVERT_THREADS, 0, s>>>((const uint16_t*)x, (const int*)index, (uint8_t*)codes, scales, rows, source_rows, K);
            return hipGetLastError();
        }
        template <bool BF16>
        hipError_t launch_weights(hipStream_t s, const void* w, void* codes, float* scales, int matrices, int N, int K)
        {
            fp8_quantize_weights_kernel<BF16><<<matrices * blocks_of(N) * blocks_of(K), BLOCK_WAVES * WAVE, 0, s>>>((const uint16_t*)w, (uint8_t*)codes, scales, blocks_of(N), N, K);
            return hipGetLastError();
        }
    } // namespace

    hipError_t launch_fp8_quantize(hipStream_t s, const void* x, bool bf16, const void* index, void* codes, float* scales, int rows, int source_rows, int K)
    {
        // (up to 512 a lane of 16 would leave half of the wavefront without any)
        if (K <= 512)
            return bf16 ? launch_rows<true, 8>(s, x, index, codes, scales, rows, source_rows, K) : launch_rows<false, 8>(s, x, index, codes, scales, rows, source_rows, K);
        return bf16 ? launch_rows<true, 16>(s, x, index, codes, scales, rows, source_rows, K) : launch_rows<false, 16>(s, x, index, codes, scales, rows, source_rows, K);
    }

    hipError_t launch_fp8_quantize_weights(hipStream_t s, const void* w, bool bf16, void* codes, float* scales, int matrices, int N, int K)
    {
        return bf16 ? launch_weights<true>(s, w, codes, scales, matrices, N, K) : launch_weights<false>(s, w, codes, scales, matrices, N, K);
    }
} // namespace nnf
