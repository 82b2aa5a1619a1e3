// MXFP4 x MXFP4 in tiles through LDS, for more rows than the weights' own traffic pays for.
//
// v_mfma_scale_f32_32x32x64: lane l holds 32 values of row l % 32, one of the step's two blocks, and their scale byte.  K goes in steps
// of 256 values -- 128 bytes of a row, a whole line of memory -- and the lanes of the half g take the blocks 4 g .. 4 g + 3 of a step
// one MFMA after the other (which values meet in an MFMA is free as long as both operands agree): the four scale bytes that a lane
// needs for a step are then one aligned word, read once, its byte chosen by the instruction.
#include "mxfp4.h"
#include "mxfp4_launch.h"
#include "nnf_launch.h"

namespace nnf
{
    namespace
    {
        using namespace mx;

        constexpr int STEP_BYTES = 128; // of a row: 256 values
        constexpr int SCALE_BYTES = 16; // of a row's scale bytes: two steps, fetched together

        // WM x WN wavefronts, each with FM x 32 activation rows and FN x 32 weight rows.  LDS: two steps of codes, three pairs of steps of
        // scale bytes (half of a pair is fetched with each step, a pair ahead).
        template <int WM_, int WN_, int FM_, int FN_>
        struct Tile
        {
            static constexpr int WM = WM_, WN = WN_, FM = FM_, FN = FN_;
            static constexpr int WAVES = WM * WN, ROWS = WM * FM * 32, COLS = WN * FN * 32;
            static constexpr int STAGE = (ROWS + COLS) * STEP_BYTES;
            static constexpr int SCALES = (ROWS + COLS) * SCALE_BYTES;
            static constexpr int LOADS = (ROWS + COLS) / 8 / WAVES;           // of codes, a step and wavefront
            static constexpr int SCALE_LOADS = (ROWS + COLS) / 64;            // a pair of steps
            static constexpr int HALF_SCALE_LOADS = (SCALE_LOADS + 1) / 2;    // a step, one to a wavefront
            static constexpr int LDS = 2 * STAGE + 3 * SCALES;
            static_assert((ROWS + COLS) / 8 % WAVES == 0 && COLS % 64 == 0 && ROWS % 64 == 0 && HALF_SCALE_LOADS <= WAVES, "whole loads");
        };

        template <int OFFSET>
        __device__ __forceinline__ void lds_read_b32_nowait(uint32_t& dst, uint32_t addr)
        {
            asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(dst) : "v"(addr), "n"(OFFSET) : "memory");
        }
        __device__ __forceinline__ void load_to_lds(const uint8_t* base, uint32_t offset, uint32_t lds)
        {
            __builtin_amdgcn_global_load_lds((const void __attribute__((address_space(1)))*)(base + offset),
                                             (void __attribute__((address_space(3)))*)lds, 16, 0, 0);
        }

        template <class T, bool GATE>
        __global__ __launch_bounds__(T::WAVES* WAVE, 1) void mxfp4_tile_kernel(Operands o, int col_tiles)
        {
            extern __shared__ __align__(256) uint8_t lds[];
            const int lane = threadIdx.x & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
            const int tile = xcd_order(blockIdx.x, gridDim.x);
            const int block = tile / col_tiles;
            RowBlock rows;
            if (!find_rows(o, block, T::ROWS == 256 ? 8 : T::ROWS == 128 ? 7 : 6, rows))
                return;
            constexpr int OUT = GATE ? T::COLS / 2 : T::COLS; // columns of Y
            const int n0 = (tile - block * col_tiles) * OUT;
            const int row_bytes = o.K >> 1, scale_stride = mx_scale_stride(o.K);
            const int steps = (row_bytes + STEP_BYTES - 1) / STEP_BYTES;
            const size_t w_row = (size_t)rows.expert * (GATE ? 2 * o.N : o.N) + n0;

            // ---- what this wavefront fetches: rows of the tile in memory order, weights first, eight to a load
            // row `i` of the tile's weight rows: with SiLU-gate a wavefront's columns are half gate rows, half their up rows
            const auto weight_row = [&](int i, bool& up) {
                up = false;
                if constexpr (GATE)
                {
                    constexpr int HALF = T::FN * 16;
                    const int in = i % (2 * HALF);
                    up = in >= HALF;
                    i = i / (2 * HALF) * HALF + in % HALF;
                }
                return min(i, o.N - 1 - n0);
            };
            const uint8_t* const a_base = o.A + (size_t)rows.first * row_bytes;
            const uint8_t* const w_base = o.W + w_row * row_bytes;
            uint32_t offset[T::LOADS];
            const auto load_base = [&](int j) {
                const int row = (wave * T::LOADS + j) * 8;
                if (row >= T::COLS)
                    return a_base;
                bool up;
                weight_row(row, up);
                return up ? w_base + (size_t)o.N * row_bytes : w_base;
            };
            // piece of a row (16 bytes) that lies at slot `lane % 8` of row `row` in LDS: XORed so that the reads of 16 rows' pieces
            // spread over all banks
            const auto piece = [&](int row) { return (lane & 7) ^ ((row >> 1) & 7); };
#pragma unroll
            for (int j = 0; j < T::LOADS; ++j)
            {
                const int row = (wave * T::LOADS + j) * 8 + (lane >> 3);
                bool up;
                const int at = row < T::COLS ? weight_row(row, up) : min(row - T::COLS, rows.end - rows.first - 1);
                offset[j] = (uint32_t)at * row_bytes + piece(row) * 16;
            }
            // this wavefront's scale bytes of either half of a pair: 64 rows, one to a lane (where there are fewer loads than wavefronts,
            // some fetch the same again)
            const uint8_t* scale_from[2];
            uint32_t scale_to[2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
            {
                const int q = min(h * T::HALF_SCALE_LOADS + wave % T::HALF_SCALE_LOADS, T::SCALE_LOADS - 1);
                const int row = q * 64 + lane;
                if (q * 64 < T::COLS)
                {
                    bool up;
                    const int at = weight_row(row, up);
                    scale_from[h] = o.Ws + (w_row + at + (up ? o.N : 0)) * scale_stride;
                }
                else
                    scale_from[h] = o.As + (size_t)(rows.first + min(row - T::COLS, rows.end - rows.first - 1)) * scale_stride;
                scale_to[h] = q * 1024;
            }
            const uint32_t lds0 = lds_address(lds);
            const int last_pair = (steps - 1) >> 1;
            const auto fetch_scales = [&](int pair, int h) {
                load_to_lds((h ? scale_from[1] : scale_from[0]) + min(pair, last_pair) * SCALE_BYTES, 0,
                            lds0 + 2 * T::STAGE + pair % 3 * T::SCALES + (h ? scale_to[1] : scale_to[0]));
            };
            // codes of a step, and half of the scale bytes of the pair of steps after the step's own.  LAST: the step may end behind the
            // rows' end: a row's last piece stands for those that are not there, and is not used
            const auto fetch = [&](int step, auto last) {
                const int k0 = step * STEP_BYTES;
                const uint32_t stage = lds0 + (step & 1) * T::STAGE;
                unroll_for<0, T::LOADS>([&](auto j) {
                    uint32_t from = offset[j];
                    if constexpr (last)
                    {
                        const int p = piece((wave * T::LOADS + j) * 8 + (lane >> 3)) * 16;
                        from += min(p, row_bytes - 16 - k0) - p;
                    }
                    load_to_lds(load_base(j) + k0, from, stage + (wave * T::LOADS + j) * 1024);
                });
                fetch_scales((step >> 1) + 1, step & 1);
            };

            // ---- what it reads from LDS
            const int r = lane & 31, g = lane >> 5;
            const int wave_n = wave % T::WN, wave_m = wave / T::WN;
            uint32_t w_at[4], a_at[4];
#pragma unroll
            for (int s = 0; s < 4; ++s)
            {
                const uint32_t in_row = r * STEP_BYTES + (((4 * g + s) ^ ((r >> 1) & 7)) << 4);
                w_at[s] = lds0 + wave_n * T::FN * 32 * STEP_BYTES + in_row;
                a_at[s] = lds0 + (T::COLS + wave_m * T::FM * 32) * STEP_BYTES + in_row;
            }
            const uint32_t ws_at = lds0 + 2 * T::STAGE + (wave_n * T::FN * 32 + r) * SCALE_BYTES + 4 * g;
            const uint32_t as_at = lds0 + 2 * T::STAGE + (T::COLS + wave_m * T::FM * 32 + r) * SCALE_BYTES + 4 * g;

            floatx16 sum[T::FN][T::FM] = {};
            uintx4 wf[2][T::FN], af[2][T::FM]; // fragments of an MFMA step and of the next
            uint32_t ws[T::FN], as[T::FM], ws_next[T::FN], as_next[T::FM];

            const auto read_scales = [&](int step) {
                const uint32_t from = (step >> 1) % 3 * T::SCALES + (step & 1) * 8;
                unroll_for<0, T::FN>([&](auto f) { lds_read_b32_nowait<f * 32 * SCALE_BYTES>(ws_next[f], ws_at + from); });
                unroll_for<0, T::FM>([&](auto f) { lds_read_b32_nowait<f * 32 * SCALE_BYTES>(as_next[f], as_at + from); });
            };
            // fragment f of an MFMA step: weights, then activations
            const auto read_fragment = [&](auto f, auto set, int s, uint32_t stage) {
                if constexpr (f < T::FN)
                    lds_read_b128_nowait<f * 32 * STEP_BYTES>(wf[set][f], w_at[s] + stage);
                else
                    lds_read_b128_nowait<(f - T::FN) * 32 * STEP_BYTES>(af[set][f - T::FN], a_at[s] + stage);
            };
            // nothing read without a wait stays in flight past the straight line of code that asked for it
            const auto landed = [&](auto set) {
                lds_wait<0>(wf[set][0]);
                unroll_for<1, T::FN>([&](auto f) { lds_wait_also(wf[set][f]); });
                unroll_for<0, T::FM>([&](auto f) { lds_wait_also(af[set][f]); });
            };
            const auto take_scales = [&] {
                unroll_for<0, T::FN>([&](auto f) { lds_wait_also(ws_next[f]); ws[f] = ws_next[f]; });
                unroll_for<0, T::FM>([&](auto f) { lds_wait_also(as_next[f]); as[f] = as_next[f]; });
            };
            using Zero = std::integral_constant<int, 0>;
            using Yes = std::true_type;
            using No = std::false_type;

            // one step; the next one's first fragments and scale bytes are read during its last MFMAs.  FETCH: ask for the codes of the
            // step after the next; LAST: that one is the last; END: this one is
            const auto body = [&](int step, auto do_fetch, auto last, auto end) {
                const uint32_t stage = (step & 1) * T::STAGE;
                const int blocks = (row_bytes - step * STEP_BYTES) >> 4; // of this step and behind it
                if constexpr (end)
                {
                    // blocks behind the rows' end: 2^0 times zeros, whatever lies there
                    const int there = min(max(blocks - 4 * g, 0), 4);
                    const uint32_t mask = there == 4 ? ~0u : (1u << (8 * there)) - 1;
#pragma unroll
                    for (int f = 0; f < T::FN; ++f)
                        ws[f] = (ws[f] & mask) | (ONES & ~mask);
#pragma unroll
                    for (int f = 0; f < T::FM; ++f)
                        as[f] = (as[f] & mask) | (ONES & ~mask);
                }
                unroll_for<0, 4>([&](auto s) {
                    constexpr int SET = s & 1;
                    using Next = std::integral_constant<int, 1 - SET>;
                    constexpr bool READS = s < 3 || !end;
                    if constexpr (end)
                    {
#pragma unroll
                        for (int f = 0; f < T::FN; ++f)
                            wf[SET][f] = 4 * g + s < blocks ? wf[SET][f] : uintx4{0, 0, 0, 0};
                    }
                    if constexpr (s == 3 && READS)
                    {
                        // every wavefront has read all of this step, all of the next has landed
                        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
                        if constexpr (do_fetch)
                            fetch(step + 2, last);
                        read_scales(step + 1);
                    }
                    unroll_for<0, T::FN * T::FM>([&](auto i) {
                        constexpr int fn = i / T::FM, fm = i % T::FM;
                        if constexpr (READS && i < T::FN + T::FM)
                            read_fragment(i, Next{}, (s + 1) & 3, s < 3 ? stage : T::STAGE - stage);
                        sum[fn][fm] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(wf[SET][fn]), operand(af[SET][fm]), sum[fn][fm], FP4, FP4,
                                                                                      s, (int)ws[fn], s, (int)as[fm]);
                        __builtin_amdgcn_sched_barrier(0);
                    });
                    if constexpr (READS)
                        landed(Next{});
                    if constexpr (s == 3 && READS)
                        take_scales();
#pragma unroll
                    for (int fn = 0; fn < T::FN; ++fn)
#pragma unroll
                        for (int fm = 0; fm < T::FM; ++fm)
                            asm volatile("" : "+a"(sum[fn][fm])); // the MFMAs stay where they are written, their sums in AGPRs
                });
            };

            fetch_scales(0, 0);
            fetch_scales(0, 1);
            fetch(0, Yes{});
            asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
            if (steps > 1)
                fetch(1, Yes{});
            read_scales(0);
            unroll_for<0, T::FN>([&](auto f) { read_fragment(f, Zero{}, 0, 0); });
            unroll_for<T::FN, T::FN + T::FM>([&](auto f) { read_fragment(f, Zero{}, 0, 0); });
            landed(Zero{});
            take_scales();
            int step = 0;
            for (; step < steps - 3; ++step)
                body(step, Yes{}, No{}, No{});
            if (steps >= 3)
                body(step++, Yes{}, Yes{}, No{});
            if (steps >= 2)
                body(step++, No{}, No{}, No{});
            body(step, No{}, No{}, Yes{});

            // ---- Y: lane l of a fragment has columns 8 (i / 4) + 4 (l / 32) + i % 4 of row l % 32.  A block of 32 rows at a time goes through
            // LDS in fp32 (a part of the wavefront's own) and leaves as whole rows, 16 bytes a lane
            constexpr int FO = GATE ? T::FN / 2 : T::FN; // fragments of columns of Y
            constexpr int PITCH = FO * 128 + 16, LANES = FO * 4, PASSES = 32 * LANES / WAVE;
            static_assert(T::WAVES * 32 * PITCH <= T::LDS && WAVE % LANES == 0, "room for the results");
            uint8_t* const mine = lds + wave * (32 * PITCH);
            const int n = n0 + wave_n * FO * 32 + lane % LANES * 8;
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
            for (int fm = 0; fm < T::FM; ++fm)
            {
#pragma unroll
                for (int fn = 0; fn < FO; ++fn)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                    {
                        floatx4 y;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                        {
                            y[i] = sum[fn][fm][q * 4 + i];
                            if constexpr (GATE)
                                y[i] = silu_gate(y[i], sum[fn + FO][fm][q * 4 + i]);
                        }
                        *reinterpret_cast<floatx4*>(mine + r * PITCH + fn * 128 + q * 32 + g * 16) = y;
                    }
#pragma unroll 1
                for (int i = 0; i < PASSES; ++i)
                {
                    const int row = i * (WAVE / LANES) + lane / LANES, m = rows.first + (wave_m * T::FM + fm) * 32 + row;
                    const floatx4* const y = reinterpret_cast<const floatx4*>(mine + row * PITCH + lane % LANES * 32);
                    if (m < rows.end && n < o.N)
                        write_eight(o, y[0], y[1], m, n);
                }
            }
        }

        template <class T, bool GATE>
        hipError_t launch(hipStream_t s, const Operands& o, int row_blocks)
        {
            static LdsGrant granted;
            const hipError_t e = allow_dynamic_lds((const void*)mxfp4_tile_kernel<T, GATE>, granted, T::LDS);
            if (e != hipSuccess)
                return e;
            constexpr int OUT = GATE ? T::COLS / 2 : T::COLS;
            const int col_tiles = (o.N + OUT - 1) / OUT;
            mxfp4_tile_kernel<T, GATE><<<(unsigned)row_blocks * col_tiles, T::WAVES * WAVE, T::LDS, s>>>(o, col_tiles);
            return hipGetLastError();
        }
    } // namespace

    hipError_t launch_mxfp4_tiles(hipStream_t s, const mx::Operands& o, int rows, int row_blocks, bool gate)
    {
        if (rows == 256)
            return gate ? launch<Tile<2, 2, 4, 4>, true>(s, o, row_blocks) : launch<Tile<2, 2, 4, 4>, false>(s, o, row_blocks);
        if (rows == 128)
            return gate ? launch<Tile<2, 2, 2, 2>, true>(s, o, row_blocks) : launch<Tile<2, 2, 2, 2>, false>(s, o, row_blocks);
        return gate ? launch<Tile<1, 4, 2, 2>, true>(s, o, row_blocks) : launch<Tile<1, 4, 2, 2>, false>(s, o, row_blocks);
    }
} // namespace nnf
