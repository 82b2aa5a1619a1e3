// Routing to experts: from logits to each token's experts and weights, and to the order in which the experts' products take the tokens.
//
// A score is softmax(l) or 1 / (1 + exp(-l)); experts are chosen by score + bias among the groups whose best one or two such sums are largest; the
// lowest index wins a tie.  LANES lanes of a wavefront have a token, V experts to a lane (expert j LANES + lane): the largest is a few
// comparisons in registers and a reduction over the lanes, k times.  Four tokens to a wavefront share the instructions of that; a token of
// its own is the shorter way where there are few.  Without a bias the order of the scores is that of the logits, which is exact.  Else
// sums are computed in fp32 first; where two that are compared lie closer than fp32 can tell (some 2^-21, a bound on both errors), the whole
// wavefront chooses again for that token in 64 bits: a choice does not depend on how exp rounds.
//
// The order is a counting sort.  A pair's place among those of its expert comes from a ballot for each bit of the expert's number inside a
// wavefront, then from the counts of the wavefronts ahead in LDS, then, in a launch of its own, from those of the workgroups ahead (16 bits
// each in the workspace).  Counts are sums of integers: the same call gives the same order, (expert, token, slot).
//
// Not bound by memory (16384 tokens over 128 experts read and write 6 MB, 1.2 us of HBM): one token is a chain of reductions, each waiting for the one
// before -- 4.9 and 5.7 us for 8 of 128 and 256 experts in a graph of 40 calls (4.0 for 4 of 60), of which a launch is 1.8, and 7.4 for 256 with sigmoid, bias and groups,
// in one wavefront: 500 cycles a round of choosing, as much as six rounds for the groups; two launches cost 7.8, 9.5 and 11.7 us for 512 tokens over 60, 128 and 256; many
// tokens are bound by the instructions of the rounds, 11.6, 16.0, 24.1, 36 and 98 us for 16384 over 60, 128, 256, 512 and 1024 (128: 11.6 us choose, 5.3 sort).
//
// The scores that become weights are computed once more, to a step of fp32: by the hardware's exp and inverse, which choosing makes do with, they would be off by
// 1.5 2^-24 |l - largest| (at most 4.3e-7 of themselves in place of 2.3e-7 for normal logits of 1.5, 2-norm 5.4e-8 either way; 1e-5 where they lie 100 apart), and
// a call 0.1 .. 0.2 us shorter.
#include "grouped_tiles.h"
#include "moe_launch.h"
#include "nnf_device.h"

namespace nnf
{
    namespace
    {
        using namespace moe;

        constexpr float LOWEST = -__builtin_inff();
        constexpr float LARGEST = 3.402823466e+38f;

        // integers in the order of the numbers (-0 counts as 0); 0 is below all of them
        __device__ __forceinline__ uint32_t key_of(float v)
        {
            const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);
            return b ^ (b >> 31 ? 0xFFFFFFFFu : 0x80000000u);
        }
        __device__ __forceinline__ uint64_t key_of(double v)
        {
            const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
            return b ^ (b >> 63 ? ~0ull : 1ull << 63);
        }
        __device__ __forceinline__ float value_of(uint32_t k) { return __builtin_bit_cast(float, k ^ (k >> 31 ? 0x80000000u : 0xFFFFFFFFu)); }
        __device__ __forceinline__ double value_of(uint64_t k) { return __builtin_bit_cast(double, k ^ (k >> 63 ? 1ull << 63 : ~0ull)); }

        template <int CTRL>
        __device__ __forceinline__ uint32_t moved(uint32_t v)
        {
            return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
        }
        template <int CTRL>
        __device__ __forceinline__ uint64_t moved(uint64_t v)
        {
            return (uint64_t)moved<CTRL>((uint32_t)(v >> 32)) << 32 | moved<CTRL>((uint32_t)v);
        }
        template <int CTRL>
        __device__ __forceinline__ float moved(float v)
        {
            return __builtin_bit_cast(float, moved<CTRL>(__builtin_bit_cast(uint32_t, v)));
        }
        template <int CTRL>
        __device__ __forceinline__ double moved(double v)
        {
            return __builtin_bit_cast(double, moved<CTRL>(__builtin_bit_cast(uint64_t, v)));
        }
        // f of what a lane and the one a quarter, or half, a wavefront away have
        template <int AWAY, class F>
        __device__ __forceinline__ uint32_t across(uint32_t v, F f)
        {
            const auto both = AWAY == 32 ? __builtin_amdgcn_permlane32_swap(v, v, false, false) : __builtin_amdgcn_permlane16_swap(v, v, false, false);
            return f((uint32_t)both[0], (uint32_t)both[1]);
        }
        template <int AWAY, class F>
        __device__ __forceinline__ float across(float v, F f)
        {
            return __builtin_bit_cast(float, across<AWAY>(__builtin_bit_cast(uint32_t, v), [&](uint32_t a, uint32_t b) {
                                          return __builtin_bit_cast(uint32_t, f(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)));
                                      }));
        }
        template <int AWAY, class F>
        __device__ __forceinline__ uint64_t across(uint64_t v, F f)
        {
            const auto pairs = [](uint32_t h) {
                return AWAY == 32 ? __builtin_amdgcn_permlane32_swap(h, h, false, false) : __builtin_amdgcn_permlane16_swap(h, h, false, false);
            };
            const auto low = pairs((uint32_t)v), high = pairs((uint32_t)(v >> 32));
            return f((uint64_t)high[0] << 32 | low[0], (uint64_t)high[1] << 32 | low[1]);
        }
        template <int AWAY, class F>
        __device__ __forceinline__ double across(double v, F f)
        {
            return __builtin_bit_cast(double, across<AWAY>(__builtin_bit_cast(uint64_t, v), [&](uint64_t a, uint64_t b) {
                                          return __builtin_bit_cast(uint64_t, f(__builtin_bit_cast(double, a), __builtin_bit_cast(double, b)));
                                      }));
        }
        // f(what another lane has) until every lane of 16 has met the others, and of 64
        template <class T, class F>
        __device__ __forceinline__ T over_16_lanes(T v, F f)
        {
            v = f(v, moved<0x128>(v)); // row_ror:8
            v = f(v, moved<0x124>(v)); // row_ror:4
            v = f(v, moved<0x122>(v)); // row_ror:2
            v = f(v, moved<0x121>(v)); // row_ror:1
            return v;
        }
        template <int LANES, class T, class F>
        __device__ __forceinline__ T over_lanes(T v, F f)
        {
            v = over_16_lanes(v, f);
            if constexpr (LANES == 64)
                v = across<32>(across<16>(v, f), f);
            return v;
        }
        __device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
        __device__ __forceinline__ uint64_t uniform(uint64_t v) { return (uint64_t)uniform((uint32_t)(v >> 32)) << 32 | uniform((uint32_t)v); }
        // the largest of a token's keys; with a token to the wavefront in scalar registers
        template <int LANES, class Key>
        __device__ __forceinline__ Key largest(Key key)
        {
            const Key most = over_lanes<LANES>(key, [](Key a, Key b) { return a > b ? a : b; });
            if constexpr (LANES == 64)
                return uniform(most);
            else
                return most;
        }
        __device__ __forceinline__ uint32_t of_lane(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }
        __device__ __forceinline__ uint64_t of_lane(uint64_t v, int lane) { return (uint64_t)of_lane((uint32_t)(v >> 32), lane) << 32 | of_lane((uint32_t)v, lane); }
        __device__ __forceinline__ uint32_t least_of_16_lanes(uint32_t v)
        {
            return over_16_lanes(v, [](uint32_t a, uint32_t b) { return min(a, b); });
        }

        __device__ __forceinline__ void lanes_meet()
        {
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }

        __device__ __forceinline__ float as_logit(float v) { return v != v ? LOWEST : fminf(v, LARGEST); }
        // logit `at`, counted from the first of token `row / E`
        __device__ __forceinline__ float logit(const Routing& r, size_t row, uint32_t at)
        {
            if (r.type == 0)
                return as_logit((float)((const half_t*)r.logits + row)[at]);
            if (r.type == 1)
                return as_logit(__builtin_bit_cast(float, (uint32_t)((const uint16_t*)r.logits + row)[at] << 16));
            return as_logit(((const float*)r.logits + row)[at]);
        }
        // the logits of the token whose first one is `from` behind `row`; behind the last one the lowest number
        template <int LANES, int V>
        __device__ __forceinline__ void logits_of(const Routing& r, size_t row, uint32_t from, float (&v)[V])
        {
            const int lane = threadIdx.x & (LANES - 1);
            int E = r.E;
            if (r.type == 2)
            {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    v[j] = ((const float*)r.logits + row)[from + min(j * LANES + lane, E - 1)];
            }
            else
            {
                uint16_t bits[V];
#pragma unroll
                for (int j = 0; j < V; ++j)
                    bits[j] = ((const uint16_t*)r.logits + row)[from + min(j * LANES + lane, E - 1)];
#pragma unroll
                for (int j = 0; j < V; ++j)
                    v[j] = r.type == 0 ? (float)__builtin_bit_cast(half_t, bits[j]) : __builtin_bit_cast(float, (uint32_t)bits[j] << 16);
            }
            asm volatile("" : "+s"(E)); // (compared again: V comparisons kept are as many pairs of scalar registers)
#pragma unroll
            for (int j = 0; j < V; ++j)
                v[j] = j * LANES + lane < E ? as_logit(v[j]) : LOWEST;
        }

        __device__ __forceinline__ float exp_of(float v) { return __expf(v); }
        __device__ __forceinline__ double exp_of(double v) { return exp(v); }
        __device__ __forceinline__ float inverse_of(float v) { return __builtin_amdgcn_rcpf(v); }
        __device__ __forceinline__ double inverse_of(double v) { return 1 / v; }

        // exp(v - top) to a step of fp32 however far apart they are: what the rounded difference lacks, times its exp, is added.  (Beyond fp32 it is not finite, and exp 0.)
        __device__ __forceinline__ float exp_of_difference(float v, float top)
        {
            const float d = v - top, t = d - v, rest = (v - (d - t)) - (top + t), e = expf(d);
            return e > 0 ? __builtin_fmaf(e, rest, e) : 0.0f;
        }

        // f(0) .. f(V - 1), four at a time (all of them at once would be registers that there are not)
        template <int V, class F>
        __device__ __forceinline__ void each(F f)
        {
            unroll_for<0, V>([&](auto j) {
                f((int)j);
                if constexpr (j % 4 == 3)
                    __builtin_amdgcn_sched_barrier(0);
            });
        }

        // The experts of the token whose logits begin `from` behind `row`: its lane p < k gets the p-th, and its score (0 of one that is masked).  room: a place
        // in LDS for E + groups values.  false: numbers that decide lie closer than Real can tell
        template <int LANES, int V, class Real, class Key>
        __device__ __forceinline__ bool choose(const Routing& r, size_t row, uint32_t from, Real* room, int& expert, Real& score)
        {
            constexpr bool APPROXIMATE = sizeof(Real) == 4;
            constexpr Real UNIT = (Real)(1.0 / (1 << 23));
            int lane = threadIdx.x & (LANES - 1);
            asm volatile("" : "+v"(lane)); // (what comes of it would be kept from turn to turn, for each of the lane's experts)
            float v[V];
            logits_of<LANES>(r, row, from, v);
            // whether a comes ahead of b whatever their errors are, of sums of `terms` scores each.  fp32: exp and the inverse are off by 2^-23 of themselves, exp's
            // argument l by 2^-24 |l| 1.5, which a score feels s (1 - s) times (at most 1/4, with |l| 0.28): two sigmoids by 4 of 2^-23.  Two softmax
            // scores, of at most 1 together, by 3 of these and by as much as their sum over 1024 experts can be, 3 more.  Sums round to 2^-24 of
            // themselves, those of two scores and biases as if they were 2 larger (see below)
            const auto sure = [&](Real a, Real b, Real terms) { return a - b > terms * (r.sigmoid ? 6 : 8) * UNIT + 2 * UNIT * (__builtin_fabs(a) + __builtin_fabs(b)); };
            bool certain = true;

            Real top = 0, sum = 1, over = 0;
            if (!r.sigmoid)
            {
                float most = v[0];
#pragma unroll
                for (int j = 1; j < V; ++j)
                    most = fmaxf(most, v[j]);
                most = over_lanes<LANES>(most, [](float a, float b) { return fmaxf(a, b); });
                top = most == LOWEST ? 0 : (Real)most;
                double all = 0; // (so that the sum adds nothing to the errors of the terms)
                each<V>([&](int j) { all += (double)exp_of((Real)v[j] - top); });
                all = over_lanes<LANES>(all, [](double a, double b) { return a + b; });
                sum = (Real)all;
                over = all > 0 ? inverse_of(sum) : 0;
            }
            const auto score_of = [&](float x) -> Real { return r.sigmoid ? inverse_of(1 + exp_of(-(Real)x)) : exp_of((Real)x - top) * over; };

            const bool restricted = r.top_groups < r.groups, by_logit = !r.bias, exact = by_logit && (!restricted || r.group_top == 1);
            const int size = r.E / r.groups;
            const uint32_t inverse = ((1u << 22) + size - 1) / size; // i / size = i inverse >> 22 for i below 1024: the excess stays below 1 / size
            int E = r.E;
            asm volatile("" : "+s"(E));
            // (one question after the other, each for all of the lane's experts: asked for each expert they are branches for each)
            Real c[V];
            if (exact)
            {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    c[j] = v[j];
            }
            else
            {
                if (r.sigmoid)
                    each<V>([&](int j) { c[j] = inverse_of(1 + exp_of(-(Real)v[j])); });
                else
                    each<V>([&](int j) { c[j] = exp_of((Real)v[j] - top) * over; });
                if (r.bias)
                    each<V>([&](int j) { c[j] += (Real)r.bias[min(j * LANES + lane, E - 1)]; });
                each<V>([&](int j) { c[j] = c[j] != c[j] || v[j] == LOWEST ? (Real)LOWEST : c[j] > (Real)LARGEST ? (Real)LARGEST : c[j]; });
            }
            if (restricted)
                each<V>([&](int j) {
                    const int i = j * LANES + lane;
                    if (i < E)
                        room[i + (i * inverse >> 22)] = c[j]; // (a group's values behind each other, a group a value further: other banks)
                });
            Key key[V];
            if (by_logit)
                each<V>([&](int j) { key[j] = j * LANES + lane < E ? key_of((Real)v[j]) : 0; });
            else
                each<V>([&](int j) { key[j] = j * LANES + lane < E ? key_of(c[j]) : 0; });
            if (restricted)
            {
                constexpr int PARTS = LANES / MAX_GROUPS; // lanes to a group
                lanes_meet();
                const int group = lane / PARTS;
                Real first = LOWEST, second = LOWEST;
                if (group < r.groups)
                    for (int i0 = lane % PARTS; i0 < size; i0 += 4 * PARTS)
                    {
                        Real some[4]; // (four reads under way at once)
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            some[u] = room[group * (size + 1) + min(i0 + u * PARTS, size - 1)];
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                        {
                            const Real x = i0 + u * PARTS < size ? some[u] : (Real)LOWEST;
                            second = x > first ? first : x > second ? x : second;
                            first = x > first ? x : first;
                        }
                    }
                if constexpr (PARTS > 1)
                {
                    static_assert(PARTS == 4, "a group's lanes are four neighbours");
                    const auto meet = [&](Real other_first, Real other_second) {
                        const Real less = first < other_first ? first : other_first;
                        first = first < other_first ? other_first : first;
                        second = second < other_second ? other_second : second;
                        second = second < less ? less : second;
                    };
                    meet(moved<0xB1>(first), moved<0xB1>(second)); // quad_perm 1,0,3,2
                    meet(moved<0x4E>(first), moved<0x4E>(second)); // 2,3,0,1
                }
                lanes_meet();
                // (large biases that cancel in a group's sum: their rounding is not in the sum's size)
                if (APPROXIMATE && r.group_top == 2)
                    certain = !__any(__builtin_fabs(first) + __builtin_fabs(second) > 4 + 2 * __builtin_fabs(first + second));
                // a group's place: how many are ahead of it, each compared with all others (a few instructions each that do not wait for one another)
                const Key group_key = group < r.groups ? key_of(r.group_top == 1 ? first : first + second) : 0;
                int place = 0;
                if constexpr (LANES == 64)
                {
#pragma unroll
                    for (int g = 0; g < MAX_GROUPS; ++g)
                    {
                        const Key other = of_lane(group_key, g * PARTS);
                        place += other > group_key || (other == group_key && g < group);
                    }
                }
                else
                {
                    Key other = group_key;
                    uint32_t whose = (uint32_t)group;
#pragma unroll
                    for (int g = 1; g < MAX_GROUPS; ++g)
                    {
                        other = moved<0x121>(other), whose = moved<0x121>(whose); // row_ror:1
                        place += other > group_key || (other == group_key && (int)whose < group);
                    }
                }
                const bool used = group < r.groups && place < r.top_groups;
                const int first_lane = threadIdx.x & (WAVE - LANES); // of the token
                using Lanes = std::conditional_t<LANES == 64, uint64_t, uint32_t>;
                const Lanes kept = (Lanes)(__ballot(used) >> first_lane);
                if (APPROXIMATE && !exact)
                {
                    // (the last that is used and any that is not: their order among themselves changes nothing)
                    const Key last = over_lanes<LANES>(used ? group_key : ~(Key)0, [](Key a, Key b) { return a < b ? a : b; });
                    const uint64_t close = __ballot(group < r.groups && !used && !sure(value_of(last), value_of(group_key), 2));
                    certain = certain && (close >> first_lane & (LANES == 64 ? ~0ull : (1ull << (LANES & 63)) - 1)) == 0;
                }
                asm volatile("" : "+v"(lane)); // (an expert's group is computed again, in the place of V registers)
                each<V>([&](int j) {
                    if (!(kept >> ((uint32_t)(j * LANES + lane) * inverse >> 22 & 15) * PARTS & 1))
                        key[j] = 0;
                });
            }

            const int turns = r.k + (APPROXIMATE && !by_logit ? 1 : 0);
            Key last = 0, own = 0;
            expert = 0;
            for (int p = 0; p < turns; ++p)
            {
                Key most = key[0];
#pragma unroll
                for (int j = 1; j < V; ++j)
                    most = key[j] > most ? key[j] : most;
                const Key best = largest<LANES>(most);
                if (APPROXIMATE && !by_logit && p > 0 && best != 0)
                    certain = certain && sure(value_of(last), value_of(best), 1);
                last = best;
                // the lowest index that has it: of the registers the first, of the lanes the first
                int at = 0;
                if constexpr (LANES == 64)
                {
                    uint64_t has = 0;
#pragma unroll
                    for (int j = V - 1; j >= 0; --j)
                    {
                        const uint64_t m = __ballot(key[j] == best);
                        has = m ? m : has;
                        at = m ? j * WAVE : at;
                    }
                    at += __builtin_ctzll(has);
                }
                else
                {
                    uint32_t mine = ~0u;
#pragma unroll
                    for (int j = V - 1; j >= 0; --j)
                        mine = key[j] == best ? (uint32_t)(j * LANES + lane) : mine;
                    at = (int)least_of_16_lanes(mine);
                }
                if (lane == p)
                    expert = at, own = best;
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (j * LANES + lane == at)
                        key[j] = 0;
            }
            score = 0;
            if (lane < r.k && own != key_of((Real)LOWEST))
            {
                const float x = by_logit ? (float)value_of(own) : logit(r, row, from + expert);
                // (once a token, so not by the hardware's exp and inverse, which the choice makes do with)
                if constexpr (APPROXIMATE)
                    score = r.sigmoid ? 1 / (1 + expf(-x)) : exp_of_difference(x, top) / sum;
                else
                    score = score_of(x);
            }
            return certain;
        }

        // `before` of thread t's run of EACH experts: how many pairs the experts ahead have (own: its own ones').  sums: a word for each wavefront
        template <int WAVES, int EACH>
        __device__ __forceinline__ uint32_t pairs_ahead(const uint32_t (&own)[EACH], uint32_t* sums)
        {
            const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
            uint32_t all = 0;
#pragma unroll
            for (int i = 0; i < EACH; ++i)
                all += own[i];
            uint32_t before = (uint32_t)sum_up_to_lane((int)all);
            if (lane == WAVE - 1)
                sums[wave] = before;
            __syncthreads();
            before -= all;
            uint32_t ahead[WAVES];
#pragma unroll
            for (int w = 0; w < WAVES; ++w)
                ahead[w] = sums[w];
#pragma unroll
            for (int w = 0; w < WAVES; ++w)
                before += w < wave ? ahead[w] : 0;
            return before;
        }

        __device__ __forceinline__ int live_tokens(const Routing& r) { return r.live ? min(max(*r.live, 0), r.tokens) : r.tokens; }

        // the values that LDS holds for a wavefront's tokens, in the first choice and in 64 bits
        template <int LANES>
        constexpr __host__ __device__ int room_bytes(int E)
        {
            return (E + MAX_GROUPS) * (WAVE / LANES * 4 > 8 ? WAVE / LANES * 4 : 8);
        }

        // ONE: a workgroup does all, in one turn; else it leaves its counts and its pairs' places among its own to the launch that sorts
        template <int LANES, int V, int WAVES, bool ONE>
        __global__ __launch_bounds__(WAVES* WAVE) void moe_route_kernel(Routing r)
        {
            extern __shared__ __align__(16) uint8_t lds[];
            constexpr int TURN = WAVE / LANES, EACH = (MAX_EXPERTS + WAVES * WAVE - 1) / (WAVES * WAVE); // tokens of a wavefront; experts of a thread
            uint32_t* const counts = (uint32_t*)lds;        // [WAVES][E]
            uint32_t* const sums = counts + WAVES * r.E;    // [WAVES]
            uint8_t* const rooms = (uint8_t*)(sums + WAVES);
            const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x & (LANES - 1), slot = threadIdx.x % WAVE / LANES;
            const int live = live_tokens(r), bits = 32 - __builtin_clz(r.E);
            const int each = ONE ? r.tokens : tokens_of_workgroup(r.tokens);
            const int first = (int)blockIdx.x * each, end = min(first + each, r.tokens);
            uint32_t so_far[EACH] = {}; // pairs of the thread's experts in the turns before
            for (int turn = first; turn < end; turn += TURN * WAVES)
            {
                // (its own wavefront's: read by others behind the next barrier)
                for (int i = threadIdx.x & (WAVE - 1); i < r.E; i += WAVE)
                    counts[wave * r.E + i] = 0;
                lanes_meet();
                const int t0 = turn + wave * TURN, t = t0 + slot;
                const bool there = t < end && t < live;
                int expert = 0;
                float score = 0;
                if (t0 < end && t0 < live)
                {
                    // (a slot without a token looks at the last one)
                    const size_t row = (size_t)t0 * r.E;
                    const int last = min(end, live) - 1 - t0;
                    uint8_t* const room = rooms + wave * room_bytes<LANES>(r.E);
                    const bool certain = choose<LANES, V, float, uint32_t>(r, row, min(slot, last) * r.E, (float*)room + slot * (r.E + MAX_GROUPS), expert, score);
                    if (const uint64_t again = __ballot(!certain))
                        for (int s = 0; s < TURN; ++s)
                            if (again >> (s * LANES) & 1)
                            {
                                int e;
                                double x;
                                choose<64, V * LANES / 64, double, uint64_t>(r, row, min(s, last) * r.E, (double*)room, e, x);
                                const int e_here = __shfl(e, lane);
                                const float x_here = __shfl((float)x, lane);
                                expert = slot == s ? e_here : expert;
                                score = slot == s ? x_here : score;
                            }
                    if (r.renormalize)
                        score /= over_16_lanes(score, [](float a, float b) { return a + b; }) + 1e-20f;
                }
                const bool pair = there && lane < r.k;
                if (t < end && lane < r.k)
                {
                    r.weights[(size_t)t * r.k + lane] = there ? score * r.scale : 0.0f;
                    r.experts[(size_t)t * r.k + lane] = there ? expert : -1;
                }
                // the wavefront's pairs of the same expert: how many are ahead, and the last one counts them
                uint64_t peers = __ballot(pair);
                for (int b = 0; b < bits; ++b)
                {
                    const uint64_t set = __ballot(expert >> b & 1);
                    peers &= expert >> b & 1 ? set : ~set;
                }
                const int id = threadIdx.x & (WAVE - 1);
                uint32_t place = (uint32_t)__builtin_popcountll(peers & ((1ull << id) - 1));
                if (pair && peers >> id == 1)
                    counts[wave * r.E + expert] = place + 1;
                __syncthreads();
                // counts become what is ahead of a wavefront: the turns before, the wavefronts before; ONE: the experts before
                uint32_t n[EACH][WAVES], own[EACH] = {};
#pragma unroll
                for (int i = 0; i < EACH; ++i)
                {
                    const int e = (int)threadIdx.x * EACH + i;
#pragma unroll
                    for (int w = 0; w < WAVES; ++w)
                        n[i][w] = e < r.E ? counts[w * r.E + e] : 0;
#pragma unroll
                    for (int w = 0; w < WAVES; ++w)
                        own[i] += n[i][w];
                }
                uint32_t before = ONE ? pairs_ahead<WAVES>(own, sums) : 0;
#pragma unroll
                for (int i = 0; i < EACH; ++i)
                {
                    const int e = (int)threadIdx.x * EACH + i;
                    uint32_t at = ONE ? before : so_far[i];
#pragma unroll
                    for (int w = 0; w < WAVES; ++w)
                    {
                        if (e < r.E)
                            counts[w * r.E + e] = at;
                        at += n[i][w];
                    }
                    if constexpr (ONE)
                    {
                        if (e < r.E)
                            r.offsets[e] = (int)before;
                        if (e == r.E - 1)
                            r.offsets[r.E] = (int)at;
                    }
                    before += own[i];
                    so_far[i] += own[i];
                }
                __syncthreads();
                if (pair)
                {
                    place += counts[wave * r.E + expert];
                    r.positions[(size_t)t * r.k + lane] = (int)place;
                    if constexpr (ONE)
                        r.rows[place] = t;
                }
                else if (ONE && t < end && lane < r.k)
                {
                    // (tokens that are not there come behind all others, in their place as in the input)
                    r.positions[t * r.k + lane] = -1;
                    r.rows[t * r.k + lane] = -1;
                }
                if constexpr (!ONE)
                    __syncthreads();
            }
            if constexpr (!ONE)
            {
#pragma unroll
                for (int i = 0; i < EACH; ++i)
                    if (const int e = (int)threadIdx.x * EACH + i; e < r.E)
                        counts[e] = so_far[i];
                __syncthreads();
                for (int i = threadIdx.x; i < count_words(r.E); i += WAVES * WAVE)
                    r.counts[(size_t)blockIdx.x * count_words(r.E) + i] = counts[2 * i] | (2 * i + 1 < r.E ? counts[2 * i + 1] << 16 : 0);
            }
        }

        // pairs go from their place among their workgroup's to their place among all
        template <int WAVES>
        __global__ __launch_bounds__(WAVES* WAVE) void moe_sort_kernel(Routing r)
        {
            extern __shared__ __align__(16) uint8_t lds[];
            constexpr int THREADS = WAVES * WAVE, EACH = (MAX_EXPERTS + THREADS - 1) / THREADS;
            uint32_t* const total = (uint32_t*)lds;    // [E]
            uint32_t* const ahead = total + r.E;       // [E]: of the workgroups before; then with the experts before
            uint32_t* const sums = ahead + r.E;        // [WAVES]
            for (int i = threadIdx.x; i < 2 * r.E; i += THREADS)
                total[i] = 0;
            const int each = tokens_of_workgroup(r.tokens), begin = (int)blockIdx.x * each * r.k, end = min(((int)blockIdx.x + 1) * each, r.tokens) * r.k;
            // (the first pair of a thread is asked for ahead of all else)
            const int p0 = begin + (int)threadIdx.x;
            int expert = p0 < end ? r.experts[p0] : -1, place = p0 < end ? r.positions[p0] : 0;
            __syncthreads();
            // everybody's counts: a thread has a word of some of the rows, a run of loads at a time
            const int words = count_words(r.E), groups = (int)gridDim.x;
            const int parts = max(THREADS / words, 1), part = threadIdx.x / words;
            if (part < parts)
                for (int w = threadIdx.x % words; w < words; w += THREADS)
                {
                    uint32_t all[2] = {0, 0}, before[2] = {0, 0};
                    constexpr int RUN = 16;
                    for (int g0 = part; g0 < groups; g0 += parts * RUN)
                    {
                        uint32_t c[RUN];
#pragma unroll
                        for (int i = 0; i < RUN; ++i)
                            c[i] = r.counts[(size_t)min(g0 + i * parts, groups - 1) * words + w];
#pragma unroll
                        for (int i = 0; i < RUN; ++i)
                        {
                            const int g = g0 + i * parts;
                            const uint32_t n = g < groups ? c[i] : 0, b = g < (int)blockIdx.x ? n : 0;
                            all[0] += n & 0xFFFF, all[1] += n >> 16;
                            before[0] += b & 0xFFFF, before[1] += b >> 16;
                        }
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (2 * w + h < r.E)
                        {
                            atomicAdd(&total[2 * w + h], all[h]);
                            atomicAdd(&ahead[2 * w + h], before[h]);
                        }
                }
            __syncthreads();
            uint32_t own[EACH];
#pragma unroll
            for (int i = 0; i < EACH; ++i)
            {
                const int e = (int)threadIdx.x * EACH + i;
                own[i] = e < r.E ? total[e] : 0;
            }
            uint32_t before = pairs_ahead<WAVES>(own, sums);
#pragma unroll
            for (int i = 0; i < EACH; ++i)
            {
                const int e = (int)threadIdx.x * EACH + i;
                if (e < r.E)
                {
                    ahead[e] += before;
                    if (blockIdx.x == 0)
                        r.offsets[e] = (int)before;
                }
                before += own[i];
                if (blockIdx.x == 0 && e == r.E - 1)
                    r.offsets[r.E] = (int)before;
            }
            __syncthreads();
            for (int p = p0; p < end; p += THREADS)
            {
                if (p != p0)
                    expert = r.experts[p], place = r.positions[p];
                // (tokens that are not there come behind all others, in their place as in the input)
                // -- inside the buffer also where another call has written to the same workspace meanwhile
                const int at = expert < 0 ? p : (int)min((uint32_t)place + ahead[min(expert, r.E - 1)], (uint32_t)(r.tokens * r.k - 1));
                r.positions[p] = expert < 0 ? -1 : at;
                r.rows[at] = expert < 0 ? -1 : p / r.k;
            }
        }

        template <int LANES, int V, int WAVES, bool ONE>
        hipError_t launch(hipStream_t s, const Routing& r)
        {
            const int bytes = (WAVES * r.E + WAVES) * 4 + (r.top_groups < r.groups ? WAVES * room_bytes<LANES>(r.E) : 0);
            static LdsGrant granted;
            const hipError_t e = allow_dynamic_lds((const void*)moe_route_kernel<LANES, V, WAVES, ONE>, granted, bytes);
            if (e != hipSuccess)
                return e;
            moe_route_kernel<LANES, V, WAVES, ONE><<<ONE ? 1 : workgroups(r.tokens), WAVES * WAVE, bytes, s>>>(r);
            return hipGetLastError();
        }
        template <int LANES, int V, int WAVES>
        hipError_t launch_both(hipStream_t s, const Routing& r)
        {
            const hipError_t e = launch<LANES, V, WAVES, false>(s, r);
            if (e != hipSuccess)
                return e;
            // a wavefront for each 64 pairs of a workgroup, up to 16: these have all counts of 128 experts under way at once
            const int pairs = tokens_of_workgroup(r.tokens) * r.k, bytes = (2 * r.E + 16) * 4;
            if (pairs <= 4 * WAVE)
                moe_sort_kernel<4><<<workgroups(r.tokens), 4 * WAVE, bytes, s>>>(r);
            else
                moe_sort_kernel<16><<<workgroups(r.tokens), 16 * WAVE, bytes, s>>>(r);
            return hipGetLastError();
        }
        // V: experts of a lane where four tokens share a wavefront
        template <int V>
        hipError_t launch_any(hipStream_t s, const Routing& r)
        {
            const int each = tokens_of_workgroup(r.tokens);
            // (a workgroup starts when its last wavefront does: 1.4 us later with 16 of them than with four)
            if (r.tokens <= 4)
                return launch<64, V / 4, 4, true>(s, r);
            if (r.tokens <= ONE_LAUNCH)
                return launch<64, V / 4, 16, true>(s, r);
            // a token to a wavefront as long as one turn of the workgroup takes them all
            if (each <= 4)
                return launch_both<64, V / 4, 4>(s, r);
            if (each <= 16)
                return launch_both<64, V / 4, 16>(s, r);
            return launch_both<16, V, V == 16 ? 8 : 16>(s, r);
        }
    } // namespace

    hipError_t launch_moe_route(hipStream_t s, const moe::Routing& r)
    {
        if (r.E <= 64)
            return launch_any<4>(s, r);
        if (r.E <= 128)
            return launch_any<8>(s, r);
        if (r.E <= 256)
            return launch_any<16>(s, r);
        // (registers for more experts of a lane, and LDS for their counts, there are of fewer wavefronts)
        if (r.E > 512)
            return r.tokens <= ONE_LAUNCH_WIDE ? launch<64, 16, 8, true>(s, r) : launch_both<64, 16, 8>(s, r);
        if (r.tokens <= ONE_LAUNCH_WIDE)
            return launch<64, 8, 8, true>(s, r);
        // (16384 tokens over 512: 41 us, and 71 with a token to a wavefront; over 1024 four would have 64 experts to a lane: 86 and 98, with bias and groups 196 and
        // 198, but 90 and 86 for 4096)
        return tokens_of_workgroup(r.tokens) <= 8 ? launch_both<64, 8, 8>(s, r) : launch_both<16, 32, 8>(s, r);
    }
} // namespace nnf
