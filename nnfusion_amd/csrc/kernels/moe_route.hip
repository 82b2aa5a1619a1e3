// Routing to experts: from logits to each token's experts and weights, and to the order in which the experts' products take the tokens.
//
// A score is softmax(l) or 1 / (1 + exp(-l)); experts are chosen by score + bias among the groups whose best one or two such sums are largest; the
// lowest index wins a tie.  Several tokens share a wavefront, LANES lanes each, V experts to a lane (expert j LANES + lane): the largest of
// a token is a few comparisons in registers and a reduction over its lanes, k times.  Without a bias the order of the scores is that of the
// logits, which is exact.  Else sums are computed in fp32 first; where two that are compared lie closer than fp32 can tell (2^-20, a bound on
// both errors), the wavefront chooses again in 64 bits: a choice does not depend on how exp rounds.
//
// The order is a counting sort: how many of each expert come from the workgroups and wavefronts ahead (counts in LDS, 16 bits each in the
// workspace between two launches), then each wavefront goes through its pairs 64 at a time, equal experts found by a ballot for each bit of
// their number.  Counts are sums of integers: the same call gives the same order, (expert, token, slot).
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
        // f(what another lane has) until every lane of the token has met all of them
        template <int LANES, class T, class F>
        __device__ __forceinline__ T over_lanes(T v, F f)
        {
            v = f(v, moved<0x128>(v)); // row_ror:8
            v = f(v, moved<0x124>(v)); // row_ror:4
            v = f(v, moved<0x122>(v)); // row_ror:2
            v = f(v, moved<0x121>(v)); // row_ror:1
            if constexpr (LANES == 64)
            {
                v = f(v, __shfl_xor(v, 16));
                v = f(v, __shfl_xor(v, 32));
            }
            return v;
        }
        // the largest key of a token's lanes and the lowest index that has it
        template <int LANES, class Key>
        __device__ __forceinline__ void best_of_lanes(Key& key, int& index)
        {
            const Key top = over_lanes<LANES>(key, [](Key a, Key b) { return a > b ? a : b; });
            const uint32_t mine = key == top ? (uint32_t)index : ~0u;
            index = (int)over_lanes<LANES>(mine, [](uint32_t a, uint32_t b) { return min(a, b); });
            key = top;
        }

        __device__ __forceinline__ void lanes_meet()
        {
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }

        __device__ __forceinline__ float logit(const Routing& r, size_t at)
        {
            float v;
            if (r.type == 0)
                v = (float)((const half_t*)r.logits)[at];
            else if (r.type == 1)
                v = __builtin_bit_cast(float, (uint32_t)((const uint16_t*)r.logits)[at] << 16);
            else
                v = ((const float*)r.logits)[at];
            return v != v ? LOWEST : fminf(v, LARGEST);
        }
        __device__ __forceinline__ float exp_of(float v) { return expf(v); }
        __device__ __forceinline__ double exp_of(double v) { return exp(v); }

        // The experts of a token, its logits in v: lane p < k gets the p-th, and its score (0 of one that is masked).  room: E + groups values
        // in LDS.  false: numbers that decide lie closer than Real can tell
        template <int LANES, int V, class Real, class Key>
        __device__ __forceinline__ bool choose(const Routing& r, const float (&v)[V], size_t row, int lane, Real* room, int& expert, Real& score)
        {
            constexpr bool APPROXIMATE = sizeof(Real) == 4;
            constexpr Real UNIT = (Real)(1.0 / (1 << 20));
            // whether a comes ahead of b whatever their errors are (of sums: 2 of them each)
            const auto sure = [&](Real a, Real b, Real errors) { return a - b > errors * UNIT * (1 + __builtin_fabs(a) + __builtin_fabs(b)); };
            bool certain = true;

            Real top = 0, sum = 0;
            if (!r.sigmoid)
            {
                float most = v[0];
#pragma unroll
                for (int j = 1; j < V; ++j)
                    most = fmaxf(most, v[j]);
                most = over_lanes<LANES>(most, [](float a, float b) { return fmaxf(a, b); });
                top = most == LOWEST ? 0 : (Real)most;
                double all = 0; // (so that the sum adds nothing to the errors of the terms)
#pragma unroll
                for (int j = 0; j < V; ++j)
                    all += (double)exp_of((Real)v[j] - top);
                sum = (Real)over_lanes<LANES>(all, [](double a, double b) { return a + b; });
            }
            const auto score_of = [&](float x) -> Real {
                if (r.sigmoid)
                    return 1 / (1 + exp_of(-(Real)x));
                return sum > 0 ? exp_of((Real)x - top) / sum : 0;
            };

            const bool restricted = r.top_groups < r.groups, by_logit = !r.bias, exact = by_logit && (!restricted || r.group_top == 1);
            const int size = r.E / r.groups;
            const uint32_t inverse = ((1u << 22) + size - 1) / size; // i / size = i inverse >> 22 for i below 1024: the excess stays below 1 / size
            Key key[V];
#pragma unroll
            for (int j = 0; j < V; ++j)
            {
                const int i = j * LANES + lane;
                Real c = v[j];
                if (!exact && v[j] != LOWEST)
                {
                    c = score_of(v[j]);
                    if (r.bias && i < r.E)
                        c += (Real)r.bias[i];
                    c = c != c ? (Real)LOWEST : c > (Real)LARGEST ? (Real)LARGEST : c;
                }
                key[j] = i < r.E ? key_of(by_logit ? (Real)v[j] : c) : 0;
                if (restricted && i < r.E)
                    room[i + (i * inverse >> 22)] = c; // (a group's values behind each other, a group a value further: other banks)
            }
            if (restricted)
            {
                lanes_meet();
                Key group_key = 0;
                if (lane < r.groups)
                {
                    const Real* const at = room + lane * (size + 1);
                    Real first = LOWEST, second = LOWEST;
                    for (int i = 0; i < size; ++i)
                    {
                        const Real c = at[i];
                        second = c > first ? first : c > second ? c : second;
                        first = c > first ? c : first;
                    }
                    group_key = key_of(r.group_top == 1 ? first : first + second);
                }
                lanes_meet();
                uint32_t kept = 0;
                Key last = 0;
                for (int g = 0; g <= r.top_groups; ++g)
                {
                    Key best = group_key;
                    int at = lane;
                    best_of_lanes<LANES>(best, at);
                    if (APPROXIMATE && !exact && g > 0)
                        certain = certain && sure(value_of(last), value_of(best), 2);
                    last = best;
                    if (g < r.top_groups)
                        kept |= 1u << at;
                    if (lane == at)
                        group_key = 0;
                }
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (!(kept >> ((uint32_t)(j * LANES + lane) * inverse >> 22 & 31) & 1))
                        key[j] = 0;
            }

            const int turns = r.k + (APPROXIMATE && !by_logit ? 1 : 0);
            Key last = 0, own = 0;
            expert = 0;
            for (int p = 0; p < turns; ++p)
            {
                Key best = key[0];
                int at = lane;
#pragma unroll
                for (int j = 1; j < V; ++j)
                    if (key[j] > best)
                        best = key[j], at = j * LANES + lane;
                best_of_lanes<LANES>(best, at);
                if (APPROXIMATE && !by_logit && p > 0 && best != 0)
                    certain = certain && sure(value_of(last), value_of(best), 1);
                last = best;
                if (lane == p)
                    expert = at, own = best;
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (at == j * LANES + lane)
                        key[j] = 0;
            }
            score = 0;
            if (lane < r.k && own != key_of((Real)LOWEST))
                score = score_of(logit(r, row + expert));
            return certain;
        }

        // A workgroup's counts, [WAVES][E], become where each wavefront's next pair of an expert goes; `total` and `ahead` [E] hold how many
        // there are of each and how many of them the workgroups ahead have.  sums: a word for each wavefront
        template <int WAVES>
        __device__ __forceinline__ void find_places(const Routing& r, uint32_t* counts, const uint32_t* total, const uint32_t* ahead, uint32_t* sums, bool writes)
        {
            constexpr int THREADS = WAVES * WAVE, EACH = (MAX_EXPERTS + THREADS - 1) / THREADS;
            const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
            uint32_t own[EACH], all = 0;
#pragma unroll
            for (int i = 0; i < EACH; ++i)
            {
                const int e = (int)threadIdx.x * EACH + i;
                own[i] = e < r.E ? total[e] : 0;
                all += own[i];
            }
            uint32_t before = all;
#pragma unroll
            for (int step = 1; step < WAVE; step *= 2)
            {
                const uint32_t other = __shfl_up(before, step);
                before += lane >= step ? other : 0;
            }
            if (lane == WAVE - 1)
                sums[wave] = before;
            __syncthreads();
            before -= all;
            for (int w = 0; w < wave; ++w)
                before += sums[w];
#pragma unroll
            for (int i = 0; i < EACH; ++i)
            {
                const int e = (int)threadIdx.x * EACH + i;
                if (e < r.E)
                {
                    if (writes)
                        r.offsets[e] = (int)before;
                    uint32_t at = before + ahead[e];
                    for (int w = 0; w < WAVES; ++w)
                    {
                        const uint32_t n = counts[w * r.E + e];
                        counts[w * r.E + e] = at;
                        at += n;
                    }
                    before += own[i];
                    if (writes && e == r.E - 1)
                        r.offsets[r.E] = (int)before;
                }
            }
            __syncthreads();
        }

        // the pairs [first, end) of a wavefront to their places; next: where its next pair of each expert goes
        template <class Expert>
        __device__ __forceinline__ void place_pairs(const Routing& r, int first, int end, uint32_t* next, Expert expert_of)
        {
            const int lane = threadIdx.x & (WAVE - 1), bits = 32 - __builtin_clz(r.E);
            for (int at = first; at < end; at += WAVE)
            {
                const int p = at + lane;
                const int e = p < end ? expert_of(p) : -1;
                uint64_t peers = __ballot(e >= 0);
                for (int b = 0; b < bits; ++b)
                {
                    const uint64_t set = __ballot(e >> b & 1);
                    peers &= e >> b & 1 ? set : ~set;
                }
                if (e >= 0)
                {
                    const uint32_t place = next[e] + (uint32_t)__builtin_popcountll(peers & ((1ull << lane) - 1));
                    r.positions[p] = (int)place;
                    r.rows[place] = p / r.k;
                    lanes_meet();
                    if (peers >> lane == 1) // the last of them
                        next[e] = place + 1;
                }
                else if (p < end)
                {
                    // (tokens that are not there come behind all others, in their place as in the input)
                    r.positions[p] = -1;
                    r.rows[p] = -1;
                }
                lanes_meet();
            }
        }

        __device__ __forceinline__ int live_tokens(const Routing& r) { return r.live ? min(max(*r.live, 0), r.tokens) : r.tokens; }

        // ONE: a workgroup does all, its wavefronts a run of tokens each; else it counts its own for the launch that sorts
        template <int LANES, int V, int WAVES, bool ONE>
        __global__ __launch_bounds__(WAVES* WAVE) void moe_route_kernel(Routing r)
        {
            extern __shared__ __align__(16) uint8_t lds[];
            constexpr int TURN = WAVE / LANES; // tokens of a wavefront at a time
            uint32_t* const counts = (uint32_t*)lds;                      // [ONE ? WAVES : 1][E]
            uint32_t* const total = counts + (ONE ? WAVES : 1) * r.E;     // [E], zeros [E] (ONE)
            uint32_t* const sums = total + (ONE ? 2 * r.E : 0);           // [WAVES]
            uint16_t* const ids = (uint16_t*)(sums + WAVES);              // [ONE_LAUNCH * MAX_K] (ONE)
            double* const rooms = (double*)(lds + (((uint8_t*)(ids + (ONE ? ONE_LAUNCH * MAX_K : 0)) - lds + 7) & ~7));
            const int wave = threadIdx.x / WAVE, lane = threadIdx.x & (LANES - 1), slot = threadIdx.x % WAVE / LANES;
            for (int i = threadIdx.x; i < (ONE ? WAVES + 2 : 1) * r.E; i += WAVES * WAVE)
                counts[i] = 0;
            __syncthreads();

            const int live = live_tokens(r);
            const int each = ONE ? (r.tokens + WAVES - 1) / WAVES : tokens_of_workgroup(r.tokens);
            // ONE: the wavefront's own run; else the workgroup's, its wavefronts in turn
            const int first = (ONE ? wave : (int)blockIdx.x) * each, end = min(first + each, r.tokens);
            for (int t0 = first + (ONE ? 0 : wave * TURN); t0 < end; t0 += ONE ? TURN : TURN * WAVES)
            {
                const int t = min(t0 + slot, end - 1);
                const bool mine = t0 + slot < end, there = t < live;
                const size_t row = (size_t)t * r.E;
                float v[V];
#pragma unroll
                for (int j = 0; j < V; ++j)
                    v[j] = j * LANES + lane < r.E ? logit(r, row + j * LANES + lane) : LOWEST;
                double* const room = rooms + (wave * TURN + slot) * (r.E + r.groups);
                int expert;
                float score;
                if (__any(!choose<LANES, V, float, uint32_t>(r, v, row, lane, (float*)room, expert, score)))
                {
                    double s;
                    choose<LANES, V, double, uint64_t>(r, v, row, lane, room, expert, s);
                    score = (float)s;
                }
                if (r.renormalize)
                    score /= over_lanes<16>(score, [](float a, float b) { return a + b; }) + 1e-20f;
                if (mine && lane < r.k)
                {
                    r.weights[(size_t)t * r.k + lane] = there ? score * r.scale : 0.0f;
                    r.experts[(size_t)t * r.k + lane] = there ? expert : -1;
                    if (there)
                        atomicAdd(&counts[(ONE ? wave : 0) * r.E + expert], 1u);
                    if constexpr (ONE)
                    {
                        ids[t * r.k + lane] = (uint16_t)(there ? expert : 0xFFFF);
                        if (there)
                            atomicAdd(&total[expert], 1u);
                    }
                }
            }
            __syncthreads();
            if constexpr (ONE)
            {
                find_places<WAVES>(r, counts, total, total + r.E, sums, true);
                place_pairs(r, first * r.k, end * r.k, counts + wave * r.E, [&](int p) { return ids[p] == 0xFFFF ? -1 : (int)ids[p]; });
            }
            else
                for (int i = threadIdx.x; i < count_words(r.E); i += WAVES * WAVE)
                    r.counts[(size_t)blockIdx.x * count_words(r.E) + i] = counts[2 * i] | (2 * i + 1 < r.E ? counts[2 * i + 1] << 16 : 0);
        }

        template <int WAVES>
        __global__ __launch_bounds__(WAVES* WAVE) void moe_sort_kernel(Routing r)
        {
            extern __shared__ __align__(16) uint8_t lds[];
            constexpr int THREADS = WAVES * WAVE;
            uint32_t* const counts = (uint32_t*)lds;           // [WAVES][E]
            uint32_t* const total = counts + WAVES * r.E;      // [E]
            uint32_t* const ahead = total + r.E;               // [E]
            uint32_t* const sums = ahead + r.E;                // [WAVES]
            const int wave = threadIdx.x / WAVE, lane = threadIdx.x & (WAVE - 1);
            for (int i = threadIdx.x; i < (WAVES + 2) * r.E; i += THREADS)
                counts[i] = 0;
            __syncthreads();
            // a wavefront's run of pairs, counted
            const int each = tokens_of_workgroup(r.tokens), end = min(((int)blockIdx.x + 1) * each, r.tokens) * r.k;
            const int run = (each * r.k + WAVES - 1) / WAVES;
            const int begin = min((int)blockIdx.x * each * r.k + wave * run, end), last = min(begin + run, end);
            for (int p = begin + lane; p < last; p += WAVE)
                if (const int e = r.experts[p]; e >= 0)
                    atomicAdd(&counts[wave * r.E + e], 1u);
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
            find_places<WAVES>(r, counts, total, ahead, sums, blockIdx.x == 0);
            place_pairs(r, begin, last, counts + wave * r.E, [&](int p) { return r.experts[p]; });
        }

        constexpr int SORT_WAVES = 4;

        template <int LANES, int V, int WAVES, bool ONE>
        hipError_t launch(hipStream_t s, const Routing& r)
        {
            const int words = (ONE ? WAVES + 2 : 1) * r.E + WAVES;
            const int ids = ONE ? ONE_LAUNCH * MAX_K * 2 : 0, rooms = r.top_groups < r.groups ? WAVES * (WAVE / LANES) * (r.E + r.groups) * 8 : 0;
            const int bytes = words * 4 + ids + 8 + rooms;
            static LdsGrant granted;
            const hipError_t e = allow_dynamic_lds((const void*)moe_route_kernel<LANES, V, WAVES, ONE>, granted, bytes);
            if (e != hipSuccess)
                return e;
            moe_route_kernel<LANES, V, WAVES, ONE><<<ONE ? 1 : workgroups(r.tokens), WAVES * WAVE, bytes, s>>>(r);
            return hipGetLastError();
        }
        template <int LANES, int V>
        hipError_t launch_either(hipStream_t s, const Routing& r)
        {
            if (r.tokens <= ONE_LAUNCH)
                return launch<LANES, V, 8, true>(s, r);
            const hipError_t e = launch<LANES, V, 4, false>(s, r);
            if (e != hipSuccess)
                return e;
            moe_sort_kernel<SORT_WAVES><<<workgroups(r.tokens), SORT_WAVES * WAVE, ((SORT_WAVES + 2) * r.E + SORT_WAVES) * 4, s>>>(r);
            return hipGetLastError();
        }
    } // namespace

    hipError_t launch_moe_route(hipStream_t s, const moe::Routing& r)
    {
        if (r.E <= 64)
            return launch_either<16, 4>(s, r);
        if (r.E <= 128)
            return launch_either<16, 8>(s, r);
        if (r.E <= 256)
            return launch_either<16, 16>(s, r);
        if (r.E <= 512)
            return launch_either<64, 8>(s, r);
        return launch_either<64, 16>(s, r);
    }
} // namespace nnf
