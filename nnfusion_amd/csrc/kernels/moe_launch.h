// Launch functions of routing and combining; nnf_api.hip checks what it is given before calling in.
#pragma once

#include "../nnf_moe_plan.h"
#include "nnf_launch.h"

namespace nnf
{
    namespace moe
    {
        struct Routing
        {
            const void* logits; // [tokens, E]
            const float* bias;  // [E] or null
            const int* live;    // the number of tokens that are there, or null: all
            float* weights;     // [tokens, k]
            int* experts;       // [tokens, k]
            int* rows;          // [tokens * k]
            int* offsets;       // [E + 1]
            int* positions;     // [tokens, k]
            uint32_t* counts;   // [workgroups, count_words(E)], unless one workgroup does all
            int tokens, E, k;
            int type;           // nnf_type
            int sigmoid, groups, top_groups, group_top, renormalize;
            float scale;
        };
    } // namespace moe

    hipError_t launch_moe_route(hipStream_t s, const moe::Routing& r);
    hipError_t launch_moe_combine(hipStream_t s, const void* x, const float* weights, const int* positions, const void* residual, void* y, int tokens,
                                  int rows, int k, int N, bool bf16);
} // namespace nnf
