// MXFP4 x MXFP4 in tiles through LDS.
//
// v_mfma_scale_f32_32x32x64: lane l holds 32 values of row l % 32, one of the step's two blocks, and their scale byte.  K goes in steps
// of 256 values -- 128 bytes of a row, a whole line of memory -- and the lanes of the half g take the blocks 4 g .. 4 g + 3 of a step
// one MFMA after the other (which values meet in an MFMA is free as long as both operands agree): the four scale bytes that a lane
// needs for a step are then one aligned word, read once, its byte chosen by the instruction.
//
// What bounds the tiles (MI355X; weights read from HBM):
//   8 .. 64 rows      HBM: 16 rows by 22016 x 4096, 49 MB, in 11.0 us (one wavefront a workgroup of 16 x 32: 688 workgroups spread evenly, 344
//                     of 16 x 64 took 12.5); 64 rows in 32 groups by 4096 x 4096 with SiLU-gate, 233 MB, in 41 .. 45 us (5.2 .. 5.7 TB/s).
//   64 .. 512 rows    a step's latencies one after the other -- a barrier, LDS, the loads into it at 64 bytes a cycle and CU --: 256 rows by
//                     4096 x 11008 on 64 x 64 in 15.4 us with the weights in the cache, 20.0 from HBM.  More steps under way (6, 8) or twice
//                     the wavefronts on half of K each: no change.
//   128 x 128         the same latencies, two workgroups a CU taking turns; HBM where groups have few rows.  1024 rows in 8 groups by 22016 x 4096
//                     with SiLU-gate, 408 MB, in 117 us (matrix cores busy 20 % of the cycles, LDS 18 %).
//   256 x 256         the clock by power, the cycles by the kernel: 4096 rows by 8192 x 8192 in 130 us (4.2 PFLOP/s) at 1.9 GHz, on zero codes the
//                     same cycles at 2.4 GHz, 92 us.  MFMAs alone would take 83 us on drawn data (6.6 PFLOP/s) and 58 on constant data (9.5):
//                     the matrix cores are busy for 55 % of the cycles, whatever the data.  What fewer cycles would give at the power limit
//                     has not been measured.  Short K: every CU loads, multiplies and stores at the same time (16000 rows in 64 groups
//                     by 4096 x 2048 in 130 us).
// Measured and not kept: lines touched ahead into L2; fragments read two MFMA steps ahead; 256 x 256 by four wavefronts of 128 x 128 (143 us,
// 134 by eight); 256 x 128 and 128 x 256 (181 us, 130 by 256 x 256; not timed on groups of about 100 rows); MFMAs at a higher wave priority
// (no change).
#include "mxfp4.h"
#include "mxfp4_launch.h"
#include "nnf_launch.h"

namespace nnf
{
    namespace
    {
        using namespace mx;

        constexpr int STEP_BYTES = 128; // of a row: 256 values
        constexpr int STEP_SCALES = 8;  // scale bytes of that

        // WK groups of WM x WN wavefronts; a group has the whole tile over its part of K, a wavefront FM x 32 activation rows and FN x 32
        // weight rows of it (ROWS below 32: that many rows of a fragment are fetched, the others repeat them).  LDS, a group: S steps of
        // codes, and scale bytes twice for G steps.  The memory pipeline's time goes by the lines that a load touches: eight rows for
        // a load of codes; the scale bytes of one step would be 8 bytes of each row and as many lines as its codes, so they are
        // fetched for G steps together, 1024 / (8 G) rows to a load.
        template <int WM_, int WN_, int WK_, int FM_, int FN_, int S_, int G_ = 4, int ROWS_ = WM_ * FM_ * 32>
        struct Tile
        {
            static constexpr int WM = WM_, WN = WN_, WK = WK_, FM = FM_, FN = FN_, S = S_, G = G_;
            static constexpr int GROUP = WM * WN, WAVES = GROUP * WK, ROWS = ROWS_, COLS = WN * FN * 32;
            static constexpr int LOADS = (ROWS + COLS) / 8 / GROUP;                         // of codes, a step and wavefront
            static constexpr int SCALE_ROWS = 1024 / (STEP_SCALES * G);                     // of a load of scale bytes
            static constexpr int ALL_SCALE_LOADS = (ROWS + COLS + SCALE_ROWS - 1) / SCALE_ROWS; // for G steps
            static constexpr int SCALE_LOADS = (ALL_SCALE_LOADS + GROUP - 1) / GROUP;       // of a wavefront
            static constexpr int STAGE = (ROWS + COLS) * STEP_BYTES, SCALES = ALL_SCALE_LOADS * 1024;
            static constexpr int GROUP_LDS = S * STAGE + 2 * SCALES;
            // a wavefront's fragments of a whole step are read together where it has few MFMAs to hide the latency of LDS behind: a step's four
            // reads one after the other took 0.26 us of 64 x 64 x 256, together 0.22 (512 x 1024 x 8192 in 12.8 and 11.3 us; with four
            // MFMAs to a read, 128 x 128, no difference: 27.2 and 27.9 us for 2048 x 4096 x 4096)
            static constexpr bool WHOLE = FM * FN <= 2;
            static constexpr int PITCH = FN * 128 + 16;                                     // fp32 results of a row of a wavefront
            static constexpr int LDS = GROUP_LDS * WK > WAVES * 32 * PITCH ? GROUP_LDS * WK : WAVES * 32 * PITCH;
            static_assert((ROWS == WM * FM * 32 || (ROWS < 32 && GROUP * FM == 1)) && (ROWS + COLS) / 8 % GROUP == 0, "whole loads");
            static_assert(LDS <= (int)MAX_LDS_BYTES && G >= S && SCALE_ROWS <= 32 && S >= 2 && (S - 1) * LOADS < 64, "room for them, and a count");
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
        // until at most N of this wavefront's loads are under way
        template <int N>
        __device__ __forceinline__ void wait_loads()
        {
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
        }

        // What lanes have written to LDS is there for the lanes that read it, and what they have read may be written over.  WK: the ranges of
        // K that meet.  One: only lanes of the same wavefront do, whose accesses LDS takes in the order of the code -- no instruction, but
        // the compiler has to keep that order
        template <int WK>
        __device__ __forceinline__ void lanes_meet()
        {
            if constexpr (WK > 1)
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            else
            {
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            }
        }

        template <class T, bool GATE>
        __global__ __launch_bounds__(T::WAVES* WAVE, 1) void mxfp4_tile_kernel(Operands o, int col_tiles)
        {
            extern __shared__ __align__(256) uint8_t lds[];
            const int lane = threadIdx.x & (WAVE - 1), wave_id = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
            const int group = wave_id / T::GROUP, wave = wave_id % T::GROUP;
            TileAt rows;
            if (!find_tile(o, blockIdx.x, T::ROWS, col_tiles, rows))
                return;
            constexpr int OUT = GATE ? T::COLS / 2 : T::COLS; // columns of Y
            const int n0 = rows.column * OUT;
            const int row_bytes = o.K >> 1, scale_stride = scale_bytes(o.K);
            const int all_steps = (row_bytes + STEP_BYTES - 1) / STEP_BYTES;
            // this group's steps: whole pairs, the same number for every group (steps behind the end add zeros)
            const int part = T::WK == 1 ? all_steps : ((all_steps + T::WK - 1) / T::WK + 1) & ~1;
            const int steps = min(part, all_steps), first_step = group * part;
            const size_t w_row = (size_t)rows.expert * (GATE ? 2 * o.N : o.N) + n0;

            // ---- what this wavefront fetches: rows of the tile in memory order, weights first, eight to a load
            // row `i` of the tile's weight rows, counted from its first: with SiLU-gate a wavefront's columns are half gate rows, half their
            // up rows
            const auto weight_row = [&](int i) {
                if constexpr (GATE)
                {
                    constexpr int HALF = T::FN * 16;
                    const int in = i % (2 * HALF);
                    return min(i / (2 * HALF) * HALF + in % HALF, o.N - 1 - n0) + (in >= HALF ? o.N : 0);
                }
                else
                    return min(i, o.N - 1 - n0);
            };
            const uint8_t* const a_base = o.A + (size_t)rows.first * row_bytes;
            const uint8_t* const w_base = o.W + w_row * row_bytes;
            uint32_t offset[T::LOADS];
            const auto load_base = [&](auto j) { return (wave * T::LOADS + (T::COLS % (T::LOADS * 8) == 0 ? 0 : (int)j)) * 8 >= T::COLS ? a_base : w_base; };
            // piece of a row (16 bytes) that lies at slot `lane % 8` of row `row` in LDS: XORed so that the reads of 16 rows' pieces
            // spread over all banks (4 cycles a read of a fragment, none of them for conflicts)
            const auto piece = [&](int row) { return (lane & 7) ^ ((row >> 1) & 7); };
#pragma unroll
            for (int j = 0; j < T::LOADS; ++j)
            {
                const int row = (wave * T::LOADS + j) * 8 + (lane >> 3);
                const int at = row < T::COLS ? weight_row(row) : min(row - T::COLS, rows.end - rows.first - 1);
                offset[j] = (uint32_t)at * row_bytes + piece(row) * 16;
            }
            // scale bytes of G steps: 16 bytes of a row to a lane, neighbouring lanes neighbouring rows (where there are fewer loads than
            // wavefronts, some fetch the same again)
            const uint8_t* scale_row[T::SCALE_LOADS];
            uint32_t scale_to[T::SCALE_LOADS];
#pragma unroll
            for (int p = 0; p < T::SCALE_LOADS; ++p)
            {
                const int q = min(p * T::GROUP + wave, T::ALL_SCALE_LOADS - 1);
                const int row = min(q * T::SCALE_ROWS + lane % T::SCALE_ROWS, T::ROWS + T::COLS - 1);
                scale_row[p] = row < T::COLS ? o.Ws + (w_row + weight_row(row)) * scale_stride
                                             : o.As + (size_t)(rows.first + min(row - T::COLS, rows.end - rows.first - 1)) * scale_stride;
                scale_to[p] = q * 1024;
            }
            const uint32_t codes_at = lds_address(lds) + group * T::GROUP_LDS, scales_at = codes_at + T::S * T::STAGE;
            const auto fetch_scales = [&](int step) {
                // (behind the end of a row: its last 16 bytes, not used)
                const int from = min((first_step + step) * STEP_SCALES + lane / T::SCALE_ROWS * 16, scale_stride - 16);
#pragma unroll
                for (int p = 0; p < T::SCALE_LOADS; ++p)
                    load_to_lds(scale_row[p] + from, 0, scales_at + (step / T::G & 1) * T::SCALES + scale_to[p]);
            };
            // codes of a step, load by load.  FULL: the step ends within
            // the rows; else a row's last piece stands for those behind its end, and is not used
            const auto fetch_load = [&](auto j, int step, uint32_t stage, auto full) {
                uint32_t from = offset[j];
                int k0 = (first_step + step) * STEP_BYTES;
                if constexpr (!full)
                {
                    k0 = min(k0, row_bytes - 16);
                    const int p = piece((wave * T::LOADS + j) * 8 + (lane >> 3)) * 16;
                    from += min(p, row_bytes - 16 - k0) - p;
                }
                else
                    asm("" : "+v"(from)); // (or the compiler keeps a 64-bit address for each load: base + offset stays an address of two parts)
                load_to_lds(load_base(j) + k0, from, codes_at + stage + (wave * T::LOADS + j) * 1024);
            };
            const auto fetch = [&](int step, uint32_t stage) {
                unroll_for<0, T::LOADS>([&](auto j) { fetch_load(j, step, stage, std::false_type{}); });
            };
            // a step that does not end within the rows, landed: what this wavefront has fetched from behind their end becomes zeros, of the
            // weights, times 2^0 of both operands
            const auto cut = [&](int step, uint32_t stage) {
                const int blocks = (row_bytes >> 4) - (first_step + step) * 8;
                unroll_for<0, T::LOADS>([&](auto j) {
                    const int row = (wave * T::LOADS + j) * 8;
                    if (row < T::COLS && piece(row + (lane >> 3)) >= blocks)
                        *reinterpret_cast<uintx4*>(lds + group * T::GROUP_LDS + stage + row * STEP_BYTES + lane * 16) = uintx4{0, 0, 0, 0};
                });
#pragma unroll
                for (int p = 0; p < T::SCALE_LOADS; ++p)
                {
                    // bytes of the step that this lane's 16 hold, if any: those behind the end
                    const int first = step % T::G * STEP_SCALES - lane / T::SCALE_ROWS * 16;
                    if (first < 0 || first >= 16)
                        continue;
                    uint32_t* const at = reinterpret_cast<uint32_t*>(lds + group * T::GROUP_LDS + T::S * T::STAGE + (step / T::G & 1) * T::SCALES + scale_to[p] + lane * 16 + first);
#pragma unroll
                    for (int d = 0; d < 2; ++d)
                    {
                        const int there = min(max(blocks - 4 * d, 0), 4);
                        const uint32_t mask = there == 4 ? ~0u : (1u << (8 * there)) - 1;
                        at[d] = (at[d] & mask) | (ONES & ~mask);
                    }
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            };
            const auto ends_outside = [&](int step) { return (first_step + step + 1) * STEP_BYTES > row_bytes; };
            constexpr int STEP_LOADS = T::LOADS;
            // until no more than `steps` steps' loads are under way (scale bytes asked for since then make it wait for more, never for less)
            const auto landed_but = [&](int steps) {
                unroll_for<1, T::S>([&](auto n) {
                    if (steps == n)
                        wait_loads<n * STEP_LOADS>();
                });
                if (steps <= 0)
                    wait_loads<0>();
            };

            // ---- what it reads from LDS
            const int r = lane & 31, g = lane >> 5;
            const int wave_n = wave % T::WN, wave_m = wave / T::WN;
            uint32_t w_at[4], a_at[4];
#pragma unroll
            for (int s = 0; s < 4; ++s)
            {
                const auto in_row = [&](int row) { return row * STEP_BYTES + (((4 * g + s) ^ ((row >> 1) & 7)) << 4); };
                w_at[s] = codes_at + wave_n * T::FN * 32 * STEP_BYTES + in_row(r);
                a_at[s] = codes_at + (T::COLS + wave_m * T::FM * 32) * STEP_BYTES + in_row(r % T::ROWS);
            }
            // (words of neighbouring rows lie 16 bytes apart, as the loads put them there, and meet four to a bank: 8 cycles a read where 2 would
            // do.  These are the conflicts that the counters show, a quarter of the cycles of LDS in the loop -- 12 of 48 a step of
            // 64 x 64, whose LDS is busy for 16 % of the time, 35 % with 256 x 256)
            const auto scale_at = [&](int row) { return scales_at + row / T::SCALE_ROWS * 1024 + row % T::SCALE_ROWS * 16 + 4 * g; };
            const uint32_t ws_at = scale_at(wave_n * T::FN * 32 + r), as_at = scale_at(T::COLS + wave_m * T::FM * 32 + r % T::ROWS);
            constexpr int FRAGMENT_SCALES = 32 / T::SCALE_ROWS * 1024; // from one fragment's scale bytes to the next one's

            floatx16 sum[T::FN][T::FM] = {};
            constexpr int U = T::WHOLE ? 4 : 1;
            uintx4 wf[2][U][T::FN], af[2][U][T::FM]; // fragments of an MFMA step (a whole step) and of the next
            uint32_t ws[T::FN], as[T::FM], ws_next[T::FN], as_next[T::FM];

            const auto read_scales = [&](int step) {
                const uint32_t from = (step / T::G & 1) * T::SCALES + step % T::G / 2 * (T::SCALE_ROWS * 16) + (step & 1) * 8;
                unroll_for<0, T::FN>([&](auto f) { lds_read_b32_nowait<f * FRAGMENT_SCALES>(ws_next[f], ws_at + from); });
                unroll_for<0, T::FM>([&](auto f) { lds_read_b32_nowait<f * FRAGMENT_SCALES>(as_next[f], as_at + from); });
            };
            // fragment f of an MFMA step: weights, then activations
            const auto read_fragment = [&](auto f, auto set, auto s, uint32_t stage) {
                constexpr int u = s % U;
                if constexpr (f < T::FN)
                    lds_read_b128_nowait<f * 32 * STEP_BYTES>(wf[set][u][f], w_at[s] + stage);
                else
                    lds_read_b128_nowait<(f - T::FN) * 32 * STEP_BYTES>(af[set][u][f - T::FN], a_at[s] + stage);
            };
            const auto read_steps = [&](auto set, uint32_t stage) {
                unroll_for<0, U>([&](auto s) { unroll_for<0, T::FN + T::FM>([&](auto f) { read_fragment(f, set, s, stage); }); });
            };
            // nothing read without a wait stays in flight past the straight line of code that asked for it
            const auto landed = [&](auto set) {
                lds_wait<0>(wf[set][0][0]);
                unroll_for<0, U>([&](auto u) {
                    unroll_for<0, T::FN>([&](auto f) { lds_wait_also(wf[set][u][f]); });
                    unroll_for<0, T::FM>([&](auto f) { lds_wait_also(af[set][u][f]); });
                });
            };
            const auto take_scales = [&] {
                unroll_for<0, T::FN>([&](auto f) { lds_wait_also(ws_next[f]); ws[f] = ws_next[f]; });
                unroll_for<0, T::FM>([&](auto f) { lds_wait_also(as_next[f]); as[f] = as_next[f]; });
            };

            fetch_scales(0);
#pragma unroll
            for (int i = 0; i < T::S; ++i)
                if (i < steps)
                    fetch(i, i * T::STAGE);
            if (ends_outside(0))
            {
                wait_loads<0>();
                cut(0, 0);
            }
            else
                landed_but(min(T::S, steps) - 1);
            if constexpr (T::GROUP > 1)
                asm volatile("s_barrier" ::: "memory");
            read_scales(0);
            read_steps(std::integral_constant<int, 0>{}, 0);
            landed(std::integral_constant<int, 0>{});
            take_scales();
            uint32_t stage = 0;
            // a step; the next one's first fragments and scale bytes are read during its last MFMAs, and what comes S steps later is asked
            // for where this one's last reads have left room.  FULL: that one ends within the rows, and its loads go out between the MFMAs
            const auto body = [&](int step, auto full) {
                const uint32_t next_stage = stage == (T::S - 1) * T::STAGE ? 0 : stage + T::STAGE;
                unroll_for<0, 4>([&](auto s) {
                    constexpr int SET = s & 1;
                    using Next = std::integral_constant<int, 1 - SET>;
                    if constexpr (s == 3)
                    {
                        // every wavefront of the group has read all of this step, all of the next has landed
                        if constexpr (full)
                            wait_loads<(T::S - 2) * STEP_LOADS>();
                        else if (step + 1 < steps && ends_outside(step + 1))
                        {
                            wait_loads<0>();
                            cut(step + 1, next_stage);
                        }
                        else
                            landed_but(min(T::S - 2, steps - 2 - step));
                        if constexpr (T::GROUP > 1)
                            asm volatile("s_barrier" ::: "memory");
                        if (step % T::G == 0 && step + T::G < steps)
                            fetch_scales(step + T::G);
                        if (!full && step + T::S < steps)
                            fetch(step + T::S, stage);
                        read_scales(step + 1);
                    }
                    // (behind the last step: what lies in LDS, not used)
                    constexpr int MFMAS = T::FN * T::FM;
                    unroll_for<0, MFMAS>([&](auto i) {
                        constexpr int fn = i / T::FM, fm = i % T::FM;
                        constexpr int READS = (T::FN + T::FM + MFMAS - 1) / MFMAS, FETCHES = (T::LOADS + MFMAS - 1) / MFMAS; // ahead of each MFMA
                        unroll_for<0, READS>([&](auto q) {
                            if constexpr (i * READS + q < T::FN + T::FM)
                                read_fragment(std::integral_constant<int, i * READS + q>{}, Next{}, std::integral_constant<int, (s + 1) & 3>{}, s < 3 ? stage : next_stage);
                        });
                        if constexpr (s == 3 && full)
                            unroll_for<0, FETCHES>([&](auto q) {
                                if constexpr (i * FETCHES + q < T::LOADS)
                                    fetch_load(std::integral_constant<int, i * FETCHES + q>{}, step + T::S, stage, std::true_type{});
                            });
                        sum[fn][fm] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(wf[SET][0][fn]), operand(af[SET][0][fm]), sum[fn][fm], FP4, FP4,
                                                                                      s, (int)ws[fn], s, (int)as[fm]);
                        __builtin_amdgcn_sched_barrier(0);
                    });
                    landed(Next{});
                    if constexpr (s == 3)
                        take_scales();
#pragma unroll
                    for (int fn = 0; fn < T::FN; ++fn)
#pragma unroll
                        for (int fm = 0; fm < T::FM; ++fm)
                            asm volatile("" : "+a"(sum[fn][fm])); // the MFMAs stay where they are written, their sums in AGPRs
                });
                stage = next_stage;
            };
            // the same with a whole step's fragments in registers: once every wavefront of the group has its own, the step's place in LDS is
            // free and the next step's fragments are read, all of them, ahead of this one's MFMAs
            const auto whole_body = [&](int step, auto set, auto full) {
                using Next = std::integral_constant<int, 1 - set>;
                const uint32_t next_stage = stage == (T::S - 1) * T::STAGE ? 0 : stage + T::STAGE;
                if constexpr (full)
                    wait_loads<(T::S - 2) * STEP_LOADS>();
                else if (step + 1 < steps && ends_outside(step + 1))
                {
                    wait_loads<0>();
                    cut(step + 1, next_stage);
                }
                else
                    landed_but(min(T::S - 2, steps - 2 - step));
                if constexpr (T::GROUP > 1)
                    asm volatile("s_barrier" ::: "memory");
                if (step % T::G == 0 && step + T::G < steps)
                    fetch_scales(step + T::G);
                if constexpr (full)
                    unroll_for<0, T::LOADS>([&](auto j) { fetch_load(j, step + T::S, stage, std::true_type{}); });
                else if (step + T::S < steps)
                    fetch(step + T::S, stage);
                read_scales(step + 1);
                read_steps(Next{}, next_stage);
                unroll_for<0, U>([&](auto s) {
                    unroll_for<0, T::FN * T::FM>([&](auto i) {
                        constexpr int fn = i / T::FM, fm = i % T::FM;
                        sum[fn][fm] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(wf[set][s][fn]), operand(af[set][s][fm]), sum[fn][fm], FP4, FP4,
                                                                                      s, (int)ws[fn], s, (int)as[fm]);
                        __builtin_amdgcn_sched_barrier(0);
                    });
                });
                landed(Next{});
                take_scales();
#pragma unroll
                for (int fn = 0; fn < T::FN; ++fn)
#pragma unroll
                    for (int fm = 0; fm < T::FM; ++fm)
                        asm volatile("" : "+a"(sum[fn][fm]));
                stage = next_stage;
            };
            int step = 0;
            const int whole = min(steps, max(row_bytes / STEP_BYTES - first_step, 0)); // steps that end within the rows
            // wavefronts whose rows all lie behind the group's end (a block of few rows in a tall tile) fetch for the others, no more: the
            // matrix cores are left to the other wavefronts of the CU
            const bool idle = T::WM > 1 && wave_m * T::FM * 32 >= rows.end - rows.first;
            if (idle)
            {
#pragma unroll 1
                for (; step < steps; ++step)
                {
                    const uint32_t next_stage = stage == (T::S - 1) * T::STAGE ? 0 : stage + T::STAGE;
                    if (step + 1 < steps && ends_outside(step + 1))
                    {
                        wait_loads<0>();
                        cut(step + 1, next_stage);
                    }
                    else
                        landed_but(min(T::S - 2, steps - 2 - step));
                    asm volatile("s_barrier" ::: "memory");
                    if (step % T::G == 0 && step + T::G < steps)
                        fetch_scales(step + T::G);
                    if (step + T::S < steps)
                        fetch(step + T::S, stage);
                    stage = next_stage;
                }
            }
            if constexpr (T::WHOLE)
            {
                using Even = std::integral_constant<int, 0>;
                using Odd = std::integral_constant<int, 1>;
#pragma unroll 1
                for (; step + 1 + T::S < whole; step += 2)
                {
                    whole_body(step, Even{}, std::true_type{});
                    whole_body(step + 1, Odd{}, std::true_type{});
                }
#pragma unroll 1
                for (; step < steps; step += 2)
                {
                    whole_body(step, Even{}, std::false_type{});
                    if (step + 1 < steps)
                        whole_body(step + 1, Odd{}, std::false_type{});
                }
            }
            else
            {
#pragma unroll 1
                for (; step + T::S < whole; ++step)
                    body(step, std::true_type{});
#pragma unroll 1
                for (; step < steps; ++step)
                    body(step, std::false_type{});
            }

            // ---- Y: lane l of a fragment has columns 8 (i / 4) + 4 (l / 32) + i % 4 of row l % 32.  A block of 32 rows at a time goes through
            // LDS in fp32; there the groups' parts are added up, in their order, and whole rows leave, 16 bytes a lane (8 cycles a write and
            // a read, 4 of the read's for conflicts: a lane reads 32 bytes in two halves)
            constexpr int MY_COLS = T::FN * (GATE ? 16 : 32); // columns of Y of a wavefront
            constexpr int LANES = MY_COLS / 8, PASSES = 32 * LANES / WAVE, MINE = (PASSES + T::WK - 1) / T::WK;
            static_assert(32 * LANES % WAVE == 0, "whole passes");
            const int n = n0 + wave_n * MY_COLS + lane % LANES * 8;
            uint8_t* const block = lds + wave * (32 * T::PITCH); // the first group's; the others' behind it
            constexpr int PART = T::GROUP * 32 * T::PITCH;
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
            for (int fm = 0; fm < T::FM; ++fm)
            {
                if (fm > 0)
                    lanes_meet<T::WK>();
#pragma unroll
                for (int fn = 0; fn < T::FN; ++fn)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<floatx4*>(block + group * PART + r * T::PITCH + fn * 128 + q * 32 + g * 16) =
                            floatx4{sum[fn][fm][q * 4], sum[fn][fm][q * 4 + 1], sum[fn][fm][q * 4 + 2], sum[fn][fm][q * 4 + 3]};
                lanes_meet<T::WK>();
                floatx4 y[MINE][2];
#pragma unroll
                for (int i = 0; i < MINE; ++i)
                {
                    const uint8_t* const at = block + ((i * T::WK + group) % PASSES * (WAVE / LANES) + lane / LANES) * T::PITCH + lane % LANES * 32;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                    {
                        y[i][h] = *reinterpret_cast<const floatx4*>(at + h * 16);
#pragma unroll
                        for (int k = 1; k < T::WK; ++k)
                            y[i][h] += *reinterpret_cast<const floatx4*>(at + k * PART + h * 16);
                        if constexpr (GATE)
                        {
                            floatx4 up = *reinterpret_cast<const floatx4*>(at + h * 16 + MY_COLS * 4);
#pragma unroll
                            for (int k = 1; k < T::WK; ++k)
                                up += *reinterpret_cast<const floatx4*>(at + k * PART + h * 16 + MY_COLS * 4);
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                y[i][h][e] = silu_gate(y[i][h][e], up[e]);
                        }
                    }
                }
                const int first = rows.first + (wave_m * T::FM + fm) * 32 + lane / LANES;
                if (n < o.N)
                    write_rows<half_t, MINE>(o, y, n, [&](int i) {
                        const int pass = i * T::WK + group, m = first + pass * (WAVE / LANES);
                        return pass < PASSES && m < rows.end && (T::ROWS >= 32 || m < rows.first + T::ROWS) ? m : -1;
                    });
            }
        }

        template <class T, bool GATE>
        hipError_t launch(hipStream_t s, const Operands& o)
        {
            static LdsGrant granted;
            const hipError_t e = allow_dynamic_lds((const void*)mxfp4_tile_kernel<T, GATE>, granted, T::LDS);
            if (e != hipSuccess)
                return e;
            const int col_tiles = column_tiles(o.N, T::COLS, GATE);
            mxfp4_tile_kernel<T, GATE><<<(unsigned)(row_blocks(o, T::ROWS) * col_tiles), T::WAVES * WAVE, T::LDS, s>>>(o, col_tiles);
            return hipGetLastError();
        }
        template <class T>
        hipError_t launch_either(hipStream_t s, const Operands& o, bool gate)
        {
            return gate ? launch<T, true>(s, o) : launch<T, false>(s, o);
        }
    } // namespace

    hipError_t launch_mxfp4_tiles(hipStream_t s, const mx::Operands& o, int kernel, bool gate)
    {
        switch (kernel)
        {
        case mx::TILE_8x32: return launch_either<Tile<1, 1, 2, 1, 1, 3, 8, 8>>(s, o, gate);
        case mx::TILE_16x32: return launch_either<Tile<1, 1, 1, 1, 1, 4, 16, 16>>(s, o, gate);
        case mx::TILE_16x32_2: return launch_either<Tile<1, 1, 2, 1, 1, 4, 8, 16>>(s, o, gate);
        case mx::TILE_16x32_4: return launch_either<Tile<1, 1, 4, 1, 1, 3, 4, 16>>(s, o, gate);
        case mx::TILE_16x64: return launch_either<Tile<1, 1, 2, 1, 2, 3, 8, 16>>(s, o, gate);
        case mx::TILE_32x64: return launch_either<Tile<1, 1, 4, 1, 2, 2>>(s, o, gate);
        case mx::TILE_32x128: return launch_either<Tile<1, 4, 1, 1, 1, 3>>(s, o, gate);
        case mx::TILE_64x64: return launch_either<Tile<2, 2, 1, 1, 1, 4>>(s, o, gate);
        case mx::TILE_64x128: return launch_either<Tile<2, 2, 1, 1, 2, 2>>(s, o, gate);
        case mx::TILE_64x128_DEEP: return launch_either<Tile<2, 2, 1, 1, 2, 4>>(s, o, gate);
        case mx::TILE_128x128: return launch_either<Tile<2, 2, 1, 2, 2, 2>>(s, o, gate);
        case mx::TILE_128x128_DEEP: return launch_either<Tile<2, 2, 1, 2, 2, 4>>(s, o, gate);
        default: return launch_either<Tile<2, 4, 1, 4, 2, 2>>(s, o, gate);
        }
    }
} // namespace nnf
