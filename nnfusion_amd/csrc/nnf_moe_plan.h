// Sizes of the routing and combining operators and how a routing is laid over workgroups: shared by the library and the emitters (host
// arithmetic only).
#pragma once

#include <stddef.h>

namespace nnf
{
    namespace moe
    {
        constexpr int MAX_EXPERTS = 1024, MAX_K = 16, MAX_GROUPS = 16;
        constexpr int MAX_PAIRS = 1 << 23; // (token, slot) pairs of a call: a workgroup's counts stay within 16 bits

        constexpr bool countable(int tokens, int k) { return tokens > 0 && k > 0 && (long long)tokens * k <= MAX_PAIRS; }
        // whether k experts can be chosen among top_groups of `groups` equal groups of E
        constexpr bool choosable(int E, int k, int groups, int top_groups, int group_top)
        {
            return E > 0 && E <= MAX_EXPERTS && k > 0 && k <= MAX_K && groups > 0 && groups <= MAX_GROUPS && E % groups == 0 && top_groups > 0 &&
                   top_groups <= groups && (group_top == 1 || group_top == 2) && group_top <= E / groups && k <= E / groups * top_groups;
        }
        constexpr bool routable(int tokens, int E, int k, int groups, int top_groups, int group_top)
        {
            return choosable(E, k, groups, top_groups, group_top) && countable(tokens, k);
        }

        // up to so many tokens one workgroup scores and sorts; above, up to MANY workgroups score, and a second launch sorts
        constexpr int ONE_LAUNCH = 16, ONE_LAUNCH_WIDE = 8, MANY = 256;
        constexpr int one_launch(int E) { return E <= 256 ? ONE_LAUNCH : ONE_LAUNCH_WIDE; }
        // (tokens up to MAX_PAIRS)
        constexpr int tokens_of_workgroup(int tokens)
        {
            const int each = (tokens + MANY - 1) / MANY;
            return (each + 3) / 4 * 4;
        }
        constexpr int workgroups(int tokens) { return (tokens + tokens_of_workgroup(tokens) - 1) / tokens_of_workgroup(tokens); }
        // a row of counts: 16 bits an expert, whole words
        constexpr int count_words(int E) { return (E + 1) / 2; }
        constexpr size_t workspace_bytes(int tokens, int E) { return tokens <= one_launch(E) ? 0 : (size_t)workgroups(tokens) * count_words(E) * 4; }

        // combining takes units of 512 columns of a token, four to a workgroup of 256 threads: fewer than 2^32 threads
        constexpr int combine_units(int N) { return (int)(((long long)N + 511) / 512); }
        constexpr bool combinable(int tokens, int k, int N) { return k <= MAX_K && (long long)tokens * combine_units(N) <= 1 << 25; }
    } // namespace moe
} // namespace nnf
