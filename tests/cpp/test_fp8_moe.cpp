// Unit tests of routing, combining and the block-scaled 8-bit operators on the host side: shape inference, what it refuses, the emitted calls, how
// a routing is laid over workgroups, and the choice of a kernel.  Prints one "PASS <name>" / "FAIL <name>: <what>" line per case.
#include "../../nnfusion_amd/csrc/nnf_fp8_plan.h"
#include "../../nnfusion_amd/csrc/nnf_moe_plan.h"
#include "nnfusion/core/operators/generic_op/generic_op.hpp"
#include "nnfusion/engine/pass/codegen/base_codegen_pass.hpp"
#include "nnfusion/engine/pass/graph/kernel_selection.hpp"

#include <cstdio>
#include <functional>
#include <set>

using namespace nnfusion;

namespace
{
    int failures = 0;
    struct Failure
    {
        std::string text;
    };
#define EXPECT(c)                                                                                                                 \
    if (!(c))                                                                                                                     \
    throw Failure{std::string(#c) + " at line " + std::to_string(__LINE__)}

    void run_case(const char* name, const std::function<void()>& f)
    {
        try
        {
            f();
            printf("PASS %s\n", name);
        }
        catch (const Failure& e)
        {
            ++failures;
            printf("FAIL %s: %s\n", name, e.text.c_str());
        }
        catch (const std::exception& e)
        {
            ++failures;
            printf("FAIL %s: %s\n", name, e.what());
        }
    }
    bool refused(const std::function<void()>& f)
    {
        try
        {
            f();
        }
        catch (const Failure&)
        {
            throw;
        }
        catch (const std::exception&)
        {
            return true;
        }
        return false;
    }

    using Node = std::shared_ptr<graph::GNode>;
    Node param(graph::Graph& g, const element::Type& t, const Shape& s)
    {
        return g.add_node_and_edge(std::make_shared<op::Parameter>(t, s), graph::GNodeVector{});
    }
    Node add(graph::Graph& g, const std::string& type, const graph::GNodeVector& in, const std::string& config = "{}")
    {
        return g.add_node_and_edge(std::make_shared<op::GenericOp>("n", type, op::OpConfig::any::parse(config)), in);
    }
    std::string emitted(const Node& n)
    {
        pass::graph::DefaultKernelSelector sel;
        auto k = sel.pick_first(n, ROCM_GPU).second;
        return k ? k->get_or_emit_source()->body_unit->get_code() : "";
    }
    bool has(const std::string& text, const std::string& part) { return text.find(part) != std::string::npos; }
} // namespace

int main()
{
    run_case("route", [] {
        graph::Graph g;
        auto l = param(g, element::f32, Shape{5, 64}), bias = param(g, element::f32, Shape{64}), tokens = param(g, element::i32, Shape{1});
        auto n = add(g, "MoeRoute", {l}, "{\"k\": 6}");
        EXPECT(n->get_output_size() == 5 && n->get_output_shape(0) == (Shape{5, 6}) && n->get_output_shape(1) == (Shape{5, 6}) && n->get_output_shape(2) == (Shape{30}) &&
               n->get_output_shape(3) == (Shape{65}) && n->get_output_shape(4) == (Shape{5, 6}));
        EXPECT(n->get_output_element_type(0) == element::f32 && n->get_output_element_type(1) == element::i32 && n->get_output_element_type(4) == element::i32);
        EXPECT(emitted(n) == "const nnf_moe_routing routing = {6, NNF_MOE_SOFTMAX, 1, 1, 1, 1, (float)1.00000000000000000e+00};\n"
                             "NNF_HIP_CHECK(nnf_moe_route(stream, input0, NNF_TYPE_F32, nullptr, nullptr, &routing, output0, output1, output2, output3, output4, 5, 64, nullptr, 0));\n");
        const auto full = emitted(add(g, "MoeRoute", {l, bias, tokens},
                                      "{\"k\": 4, \"has_bias\": true, \"has_tokens\": true, \"score\": \"sigmoid\", \"groups\": 8, \"top_groups\": 4, \"group_top\": 2, "
                                      "\"renormalize\": false, \"scale\": 2.5}"));
        EXPECT(has(full, "{4, NNF_MOE_SIGMOID, 8, 4, 2, 0, (float)2.5") && has(full, "NNF_TYPE_F32, input1, input2, &routing"));
        EXPECT(has(emitted(add(g, "MoeRoute", {param(g, element::f16, Shape{5, 64}), tokens}, "{\"k\": 4, \"has_tokens\": true}")), "NNF_TYPE_F16, nullptr, input1, &routing"));
        // many tokens: two launches, counts between them
        const auto many = emitted(add(g, "MoeRoute", {param(g, element::f32, Shape{1000, 64})}, "{\"k\": 4}"));
        EXPECT(!has(many, "nullptr, 0))") && has(many, ", " + std::to_string(nnf::moe::workspace_bytes(1000, 64)) + "))"));
        EXPECT(emitted(add(g, "MoeRoute", {param(g, element::f32, Shape{(1 << 21) + 1, 64})}, "{\"k\": 4}")).empty());
        for (const char* bad : {"{\"k\": 0}", "{\"k\": 17}", "{\"k\": 4, \"groups\": 3}", "{\"k\": 9, \"groups\": 8, \"top_groups\": 1}", "{\"k\": 2, \"groups\": 8, \"top_groups\": 9}",
                                "{\"k\": 2, \"group_top\": 3}", "{\"k\": 2, \"score\": \"tanh\"}", "{\"k\": 2, \"has_bias\": true}"})
            EXPECT(refused([&] { add(g, "MoeRoute", {l}, bad); }));
        EXPECT(refused([&] { add(g, "MoeRoute", {l, param(g, element::f32, Shape{63})}, "{\"k\": 2, \"has_bias\": true}"); }));
        EXPECT(refused([&] { add(g, "MoeRoute", {l, param(g, element::i32, Shape{2})}, "{\"k\": 2, \"has_tokens\": true}"); }));
        EXPECT(refused([&] { add(g, "MoeRoute", {param(g, element::f32, Shape{5, 1025})}, "{\"k\": 2}"); }));
        EXPECT(refused([&] { add(g, "MoeRoute", {param(g, element::i32, Shape{5, 64})}, "{\"k\": 2}"); }));
    });

    run_case("combine", [] {
        graph::Graph g;
        auto x = param(g, element::f16, Shape{30, 96}), w = param(g, element::f32, Shape{10, 3}), p = param(g, element::i32, Shape{10, 3}), r = param(g, element::f16, Shape{10, 96});
        auto n = add(g, "MoeCombine", {x, w, p});
        EXPECT(n->get_output_shape(0) == (Shape{10, 96}) && n->get_output_element_type(0) == element::f16);
        EXPECT(emitted(n) == "NNF_HIP_CHECK(nnf_moe_combine(stream, input0, input1, input2, nullptr, output0, NNF_TYPE_F16, 10, 30, 3, 96));\n");
        EXPECT(has(emitted(add(g, "MoeCombine", {x, w, p, r}, "{\"has_residual\": true}")), "input2, input3, output0"));
        EXPECT(emitted(add(g, "MoeCombine", {x, param(g, element::f32, Shape{10, 17}), param(g, element::i32, Shape{10, 17})})).empty());
        EXPECT(refused([&] { add(g, "MoeCombine", {x, w, param(g, element::i32, Shape{3, 10})}); }));
        EXPECT(refused([&] { add(g, "MoeCombine", {x, w, p, x}, "{\"has_residual\": true}"); }));
        EXPECT(refused([&] { add(g, "MoeCombine", {param(g, element::f32, Shape{30, 96}), w, p}); }));
    });

    run_case("quantize", [] {
        graph::Graph g;
        auto x = param(g, element::f16, Shape{12, 1056});
        auto n = add(g, "Fp8Quantize", {x});
        EXPECT(n->get_output_shape(0) == (Shape{12, 1056}) && n->get_output_shape(1) == (Shape{9, 12}));
        EXPECT(n->get_output_element_type(0) == element::u8 && n->get_output_element_type(1) == element::f32);
        EXPECT(emitted(n) == "NNF_HIP_CHECK(nnf_fp8_quantize(stream, input0, NNF_TYPE_F16, nullptr, output0, output1, 12, 12, 1056));\n");
        auto m = add(g, "Fp8Quantize", {x, param(g, element::i32, Shape{30})}, "{\"has_index\": true}");
        EXPECT(m->get_output_shape(0) == (Shape{30, 1056}) && has(emitted(m), "NNF_TYPE_F16, input1, output0, output1, 30, 12, 1056"));
        EXPECT(emitted(add(g, "Fp8Quantize", {param(g, element::f16, Shape{(1 << 24) + 1, 16})})).empty());
        EXPECT(refused([&] { add(g, "Fp8Quantize", {param(g, element::f16, Shape{12, 40})}); }));
        EXPECT(refused([&] { add(g, "Fp8Quantize", {param(g, element::f32, Shape{12, 64})}); }));
        EXPECT(refused([&] { add(g, "Fp8Quantize", {x, param(g, element::i64, Shape{30})}, "{\"has_index\": true}"); }));
    });

    run_case("dot", [] {
        graph::Graph g;
        auto a = param(g, element::u8, Shape{7, 528}), as = param(g, element::f32, Shape{5, 7});
        auto w = param(g, element::u8, Shape{96, 528}), ws = param(g, element::f32, Shape{1, 5});
        auto bias = param(g, element::f16, Shape{96}), residual = param(g, element::f16, Shape{7, 96});
        auto n = add(g, "Fp8Dot", {a, as, w, ws});
        EXPECT(n->get_output_shape(0) == (Shape{7, 96}) && n->get_output_element_type(0) == element::f16);
        EXPECT(emitted(n) == "NNF_HIP_CHECK(nnf_fp8_gemm(stream, input0, input1, input2, input3, output0, NNF_TYPE_F16, 7, 96, 528, nullptr, nullptr, NNF_ACT_NONE));\n");
        EXPECT(has(emitted(add(g, "Fp8Dot", {a, as, w, ws, bias, residual}, "{\"has_bias\": true, \"has_residual\": true}")), "528, input4, input5, NNF_ACT_NONE"));
        EXPECT(has(emitted(add(g, "Fp8Dot", {a, as, w, ws, residual}, "{\"has_residual\": true}")), "528, nullptr, input4, NNF_ACT_NONE"));
        // gate and up rows have blocks of their own: two rows of scales for 2 x 48 rows
        auto two = param(g, element::f32, Shape{2, 5});
        auto gate = add(g, "Fp8Dot", {a, as, w, two}, "{\"act\": \"silu_gate\"}");
        EXPECT(gate->get_output_shape(0) == (Shape{7, 48}) && has(emitted(gate), "7, 48, 528, nullptr, nullptr, NNF_ACT_SILU_GATE"));
        EXPECT(refused([&] { add(g, "Fp8Dot", {a, as, w, ws}, "{\"act\": \"silu_gate\"}"); }));
        EXPECT(refused([&] { add(g, "Fp8Dot", {a, as, w, two}); }));
        // the launcher has no gate with a bias: the node is declined, not miscompiled
        EXPECT(emitted(add(g, "Fp8Dot", {a, as, w, two, param(g, element::f16, Shape{48})}, "{\"act\": \"silu_gate\", \"has_bias\": true}")).empty());
        EXPECT(refused([&] { add(g, "Fp8Dot", {a, param(g, element::f32, Shape{7, 5}), w, ws}); }));
        EXPECT(refused([&] { add(g, "Fp8Dot", {a, as, param(g, element::u8, Shape{96, 512}), param(g, element::f32, Shape{1, 4})}); }));
        EXPECT(refused([&] { add(g, "Fp8Dot", {a, as, w, ws, param(g, element::f16, Shape{95})}, "{\"has_bias\": true}"); }));
        EXPECT(refused([&] { add(g, "Fp8Dot", {a, as, w, ws, param(g, element::f16, Shape{96, 7})}, "{\"has_residual\": true}"); }));
        EXPECT(refused([&] { add(g, "Fp8Dot", {a, as, param(g, element::u8, Shape{95, 528}), ws}, "{\"act\": \"silu_gate\"}"); }));
        EXPECT(refused([&] { add(g, "Fp8Dot", {a, as, w, ws}, "{\"act\": \"gelu\"}"); }));
        EXPECT(emitted(add(g, "Fp8Dot", {param(g, element::u8, Shape{(1 << 30) + 1, 16}), param(g, element::f32, Shape{1, (1 << 30) + 1}), param(g, element::u8, Shape{8, 16}),
                                         param(g, element::f32, Shape{1, 1})})).empty());
    });

    run_case("grouped_dot", [] {
        graph::Graph g;
        auto a = param(g, element::u8, Shape{40, 144}), as = param(g, element::f32, Shape{2, 40});
        auto w = param(g, element::u8, Shape{6, 260, 144}), ws = param(g, element::f32, Shape{6, 3, 2}), gs = param(g, element::f32, Shape{6, 4, 2});
        auto offsets = param(g, element::i32, Shape{7});
        auto n = add(g, "Fp8GroupedDot", {a, as, w, ws, offsets});
        EXPECT(n->get_output_shape(0) == (Shape{40, 260}));
        EXPECT(emitted(n) == "NNF_HIP_CHECK(nnf_fp8_grouped_gemm(stream, input0, input1, input2, input3, input4, output0, NNF_TYPE_F16, 6, 40, 260, 144, NNF_ACT_NONE));\n");
        EXPECT(has(emitted(add(g, "Fp8GroupedDot", {a, as, w, gs, offsets}, "{\"act\": \"silu_gate\"}")), "6, 40, 130, 144, NNF_ACT_SILU_GATE"));
        EXPECT(refused([&] { add(g, "Fp8GroupedDot", {a, as, w, gs, offsets}); }));
        EXPECT(refused([&] { add(g, "Fp8GroupedDot", {a, as, w, ws, param(g, element::i32, Shape{6})}); }));
        EXPECT(refused([&] { add(g, "Fp8GroupedDot", {a, as, param(g, element::u8, Shape{260, 144}), param(g, element::f32, Shape{3, 2}), offsets}); }));
    });

    // every token has a workgroup, no more of them than the counts' rows, and a workgroup's pairs fit 16 bits
    run_case("routing_over_workgroups", [] {
        using namespace nnf::moe;
        for (int tokens : {1, 17, 64, 65, 1000, 1024, 1025, 4096, 16384, 65537, 1 << 20, 1 << 23})
        {
            const int each = tokens_of_workgroup(tokens), n = workgroups(tokens);
            EXPECT(each > 0 && n > 0 && n <= MANY && (long long)n * each >= tokens && (long long)(n - 1) * each < tokens);
            for (int k : {1, 8, MAX_K})
                if ((long long)tokens * k <= MAX_PAIRS)
                    EXPECT((long long)each * k <= 65535);
            EXPECT(workspace_bytes(tokens, 60) == (tokens <= ONE_LAUNCH ? 0 : (size_t)n * 120) && workspace_bytes(tokens, 61) % 4 == 0);
        }
        EXPECT(workspace_bytes(ONE_LAUNCH_WIDE, 1024) == 0 && workspace_bytes(ONE_LAUNCH_WIDE + 1, 1024) > 0);
    });

    // no shape goes without a kernel, every kernel is some shape's, and the estimates stay finite
    run_case("choice_of_a_kernel", [] {
        using namespace nnf::fp8;
        std::set<int> seen;
        for (int experts : {0, 2, 8, 60, 128})
            for (int gate = 0; gate < 2; ++gate)
                for (int m : {1, 3, 8, 16, 17, 33, 64, 100, 129, 256, 500, 1024, 4096, 16384})
                    for (int n : {1, 64, 100, 512, 1024, 2050, 4096, 8192, 11008, 22016})
                        for (int k : {16, 96, 256, 1024, 1376, 2080, 4096, 8192, 11008, 16384})
                        {
                            const int c = choose(m, n, k, gate != 0, experts, 256);
                            EXPECT(c >= 0 && c < KERNELS && fits(FACTS[c], m, n, gate != 0, experts));
                            const float t = estimate(FACTS[c], m, n, k, gate != 0, experts, 256, bytes_of(m, n, k, gate != 0, experts));
                            EXPECT(t > 0 && t < 1e9f);
                            seen.insert(c);
                        }
        EXPECT(seen.size() == KERNELS);
        EXPECT(!fits(FACTS[TILE_16x32], 1 << 24, 4096, false, 0) && FACTS[choose(1 << 24, 4096, 32, false, 0, 256)].rows >= 128);
        EXPECT(choose(1 << 28, 1 << 12, 32, false, 0, 256) == KERNELS && !servable(1 << 28, 1 << 12, 32, false, 0));
        EXPECT(servable(1, 1 << 15, 1 << 15, true, 0) && !servable(1, 1 << 16, 1 << 15, true, 0) && servable(1, 1 << 16, 1 << 15, false, 0));
        EXPECT(convertible(1 << 24, 512) && !convertible((1 << 24) + 1, 512) && !convertible(1 << 24, 528) && convertible(1, MAX_K) && !convertible(1, MAX_K + 16) && !convertible(1, 40));
        EXPECT(weights_convertible(1, 1 << 15, 1 << 15) && !weights_convertible(1, 1 << 20, 1 << 17) && !weights_convertible(1 << 23, 128, 128) &&
               weights_convertible((1 << 23) - 1, 128, 128) && !weights_convertible(1, 128, 100));
        EXPECT(blocks_of(1) == 1 && blocks_of(128) == 1 && blocks_of(129) == 2 && blocks_of(2147483647) == 1 << 24);
    });
    return failures ? 1 : 0;
}
