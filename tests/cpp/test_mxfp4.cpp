// Unit tests of the MXFP4 operators on the host side: shape inference, what it refuses, the emitted calls, and the choice of a kernel.
// Prints one "PASS <name>" / "FAIL <name>: <what>" line per case.
#include "../../nnfusion_amd/csrc/nnf_mxfp4_plan.h"
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
    Node add(graph::Graph& g, const std::string& type, const graph::GNodeVector& in, const std::string& config = "")
    {
        return g.add_node_and_edge(std::make_shared<op::GenericOp>("n", type, config.empty() ? op::OpConfig::any() : op::OpConfig::any::parse(config)), in);
    }
    std::string emitted(const Node& n)
    {
        pass::graph::DefaultKernelSelector sel;
        auto k = sel.pick_first(n, ROCM_GPU).second;
        return k ? k->get_or_emit_source()->body_unit->get_code() : "";
    }
} // namespace

int main()
{
    run_case("quantize", [] {
        graph::Graph g;
        auto x = param(g, element::f16, Shape{12, 1056});
        auto n = add(g, "MxQuantize", {x});
        EXPECT(n->get_output_size() == 2 && n->get_output_shape(0) == (Shape{12, 528}) && n->get_output_shape(1) == (Shape{12, 48}));
        EXPECT(n->get_output_element_type(0) == element::u8 && n->get_output_element_type(1) == element::u8);
        EXPECT(emitted(n) == "NNF_HIP_CHECK(nnf_mxfp4_quantize_f16(stream, input0, nullptr, output0, output1, 12, 12, 1056));\n");
        auto m = add(g, "MxQuantize", {x, param(g, element::i32, Shape{30})}, "{\"has_index\": true}");
        EXPECT(m->get_output_shape(0) == (Shape{30, 528}) && m->get_output_shape(1) == (Shape{30, 48}));
        EXPECT(emitted(m) == "NNF_HIP_CHECK(nnf_mxfp4_quantize_f16(stream, input0, input1, output0, output1, 30, 12, 1056));\n");
        EXPECT(refused([&] { add(g, "MxQuantize", {param(g, element::f32, Shape{12, 64})}); }));
        EXPECT(refused([&] { add(g, "MxQuantize", {param(g, element::f16, Shape{12, 48})}); }));
        EXPECT(refused([&] { add(g, "MxQuantize", {param(g, element::f16, Shape{64})}); }));
        EXPECT(refused([&] { add(g, "MxQuantize", {x, param(g, element::i32, Shape{30})}); }));
        EXPECT(refused([&] { add(g, "MxQuantize", {x, param(g, element::i64, Shape{30})}, "{\"has_index\": true}"); }));
    });

    run_case("dequantize", [] {
        graph::Graph g;
        auto n = add(g, "MxDequantize", {param(g, element::u8, Shape{5, 64}), param(g, element::u8, Shape{5, 16})});
        EXPECT(n->get_output_shape(0) == (Shape{5, 128}) && n->get_output_element_type(0) == element::f16);
        EXPECT(emitted(n) == "NNF_HIP_CHECK(nnf_mxfp4_dequantize_f16(stream, input0, input1, output0, 5, 128));\n");
        EXPECT(refused([&] { add(g, "MxDequantize", {param(g, element::u8, Shape{5, 64}), param(g, element::u8, Shape{5, 4})}); }));
        EXPECT(refused([&] { add(g, "MxDequantize", {param(g, element::u8, Shape{5, 64}), param(g, element::u8, Shape{4, 16})}); }));
        EXPECT(refused([&] { add(g, "MxDequantize", {param(g, element::i8, Shape{5, 64}), param(g, element::u8, Shape{5, 16})}); }));
    });

    run_case("dot", [] {
        graph::Graph g;
        auto a = param(g, element::u8, Shape{7, 256}), as = param(g, element::u8, Shape{7, 16});
        auto w = param(g, element::u8, Shape{96, 256}), ws = param(g, element::u8, Shape{96, 16});
        auto bias = param(g, element::f16, Shape{96}), residual = param(g, element::f16, Shape{7, 96});
        auto n = add(g, "MxDot", {a, as, w, ws});
        EXPECT(n->get_output_shape(0) == (Shape{7, 96}) && n->get_output_element_type(0) == element::f16);
        EXPECT(emitted(n) == "NNF_HIP_CHECK(nnf_mxfp4_gemm(stream, input0, input1, input2, input3, output0, 7, 96, 512, nullptr, nullptr, NNF_ACT_NONE, nullptr, 0));\n");
        EXPECT(emitted(add(g, "MxDot", {a, as, w, ws, bias, residual}, "{\"has_bias\": true, \"has_residual\": true}")).find("512, input4, input5, NNF_ACT_NONE") !=
               std::string::npos);
        EXPECT(emitted(add(g, "MxDot", {a, as, w, ws, residual}, "{\"has_residual\": true}")).find("512, nullptr, input4, NNF_ACT_NONE") != std::string::npos);
        auto gate = add(g, "MxDot", {a, as, w, ws}, "{\"act\": \"silu_gate\"}");
        EXPECT(gate->get_output_shape(0) == (Shape{7, 48}) && emitted(gate).find("output0, 7, 48, 512, nullptr, nullptr, NNF_ACT_SILU_GATE") != std::string::npos);
        // the launcher has no gate with a bias: the node is declined, not miscompiled
        EXPECT(emitted(add(g, "MxDot", {a, as, w, ws, param(g, element::f16, Shape{48})}, "{\"act\": \"silu_gate\", \"has_bias\": true}")).empty());
        // nor sizes beyond its own: N * K of 2^32 with SiLU-gate, 2^30 rows of results and more
        const size_t rows = 1 << 17, k = 1 << 15;
        auto la = param(g, element::u8, Shape{4, k / 2}), las = param(g, element::u8, Shape{4, k / 32});
        auto lw = param(g, element::u8, Shape{2 * rows, k / 2}), lws = param(g, element::u8, Shape{2 * rows, k / 32});
        EXPECT(!emitted(add(g, "MxDot", {la, las, lw, lws})).empty() && emitted(add(g, "MxDot", {la, las, lw, lws}, "{\"act\": \"silu_gate\"}")).empty());
        EXPECT(emitted(add(g, "MxDot", {param(g, element::u8, Shape{(1 << 30) + 1, 16}), param(g, element::u8, Shape{(1 << 30) + 1, 16}),
                                        param(g, element::u8, Shape{8, 16}), param(g, element::u8, Shape{8, 16})})).empty());
        EXPECT(emitted(add(g, "MxQuantize", {param(g, element::f16, Shape{1 << 28, 32})})).empty());
        EXPECT(refused([&] { add(g, "MxDot", {a, as, param(g, element::u8, Shape{96, 128}), param(g, element::u8, Shape{96, 16})}); }));
        EXPECT(refused([&] { add(g, "MxDot", {a, as, w, ws, param(g, element::f16, Shape{95})}, "{\"has_bias\": true}"); }));
        EXPECT(refused([&] { add(g, "MxDot", {a, as, w, ws, param(g, element::f16, Shape{96, 7})}, "{\"has_residual\": true}"); }));
        EXPECT(refused([&] { add(g, "MxDot", {a, as, param(g, element::u8, Shape{95, 256}), param(g, element::u8, Shape{95, 16})}, "{\"act\": \"silu_gate\"}"); }));
        EXPECT(refused([&] { add(g, "MxDot", {a, as, w, ws}, "{\"act\": \"gelu\"}"); }));
    });

    run_case("grouped_dot", [] {
        graph::Graph g;
        auto a = param(g, element::u8, Shape{40, 64}), as = param(g, element::u8, Shape{40, 16});
        auto w = param(g, element::u8, Shape{6, 50, 64}), ws = param(g, element::u8, Shape{6, 50, 16}), offsets = param(g, element::i32, Shape{7});
        auto n = add(g, "MxGroupedDot", {a, as, w, ws, offsets});
        EXPECT(n->get_output_shape(0) == (Shape{40, 50}));
        EXPECT(emitted(n) == "NNF_HIP_CHECK(nnf_mxfp4_grouped_gemm(stream, input0, input1, input2, input3, input4, output0, 6, 40, 50, 128, NNF_ACT_NONE, nullptr, 0));\n");
        EXPECT(emitted(add(g, "MxGroupedDot", {a, as, w, ws, offsets}, "{\"act\": \"silu_gate\"}")).find("output0, 6, 40, 25, 128, NNF_ACT_SILU_GATE") != std::string::npos);
        EXPECT(refused([&] { add(g, "MxGroupedDot", {a, as, w, ws, param(g, element::i32, Shape{6})}); }));
        EXPECT(refused([&] { add(g, "MxGroupedDot", {a, as, w, ws, param(g, element::i64, Shape{7})}); }));
        EXPECT(refused([&] { add(g, "MxGroupedDot", {a, as, param(g, element::u8, Shape{50, 64}), param(g, element::u8, Shape{50, 16}), offsets}); }));
    });

    run_case("scale_bytes", [] {
        using namespace nnf::mx;
        EXPECT(scale_bytes(32) == 16 && scale_bytes(512) == 16 && scale_bytes(544) == 32 && scale_bytes(4096) == 128 && scale_bytes(11008) == 352);
        EXPECT(supported(32) && supported(MAX_K) && !supported(0) && !supported(-32) && !supported(48) && !supported(MAX_K + 32));
    });

    // no shape goes without a kernel, a form with SiLU-gate gets one that has it, every kernel is some shape's, and the estimates stay finite
    run_case("choice_of_a_kernel", [] {
        using namespace nnf::mx;
        std::set<int> seen;
        for (int experts : {0, 2, 8, 60, 128})
            for (int gate = 0; gate < 2; ++gate)
                for (int m : {1, 3, 8, 16, 17, 33, 64, 100, 129, 256, 500, 1024, 4096, 16384})
                    for (int n : {1, 64, 100, 512, 1024, 2050, 4096, 8192, 11008, 22016})
                        for (int k : {32, 96, 256, 1024, 1376, 2080, 4096, 8192, 11008, 16384})
                        {
                            const int c = choose(m, n, k, gate != 0, experts, 256);
                            EXPECT(c >= 0 && c < KERNELS && fits(FACTS[c], m, n, gate != 0, experts));
                            const float t = estimate(FACTS[c], m, n, k, gate != 0, experts, 256, bytes_of(m, n, k, gate != 0, experts));
                            EXPECT(t > 0 && t < 1e9f);
                            seen.insert(c);
                        }
        EXPECT(seen.size() == KERNELS);
        // a grid has fewer than 2^32 threads: where a small tile would need more, a larger one serves; where all would, none
        EXPECT(!fits(FACTS[TILE_16x64], 1 << 24, 4096, false, 0) && FACTS[choose(1 << 24, 4096, 32, false, 0, 256)].rows >= 128);
        EXPECT(choose(1 << 28, 1 << 12, 32, false, 0, 256) == KERNELS && choose(1 << 23, 1 << 16, 32, true, 1 << 23, 256) == KERNELS);
        EXPECT(convertible(1 << 28, 32) == false && convertible((1 << 28) - 16, 512) && !convertible(1 << 27, 1024) && convertible(1, MAX_K));
        // the bound on blocks of rows holds for any groups: all rows in one, spread evenly, one row each
        for (int rows : {8, 16, 64, 256})
            for (int m : {1, 7, 64, 1000})
                for (int experts : {1, 5, 64, 300})
                {
                    const long long most = most_row_blocks(m, experts, rows);
                    long long even = 0;
                    for (int e = 0; e < experts; ++e)
                        even += (m / experts + (e < m % experts) + rows - 1) / rows;
                    const int ones = experts - 1 < m - 1 ? experts - 1 : m - 1;
                    EXPECT(most >= (m + rows - 1) / rows && most >= even && most >= ones + (m - ones + rows - 1) / rows && most <= m);
                }
    });

    // a node gets a kernel where the call has one: not where every tile would need a larger grid than there is
    run_case("nodes_beyond_every_grid", [] {
        using namespace nnf::mx;
        graph::Graph g;
        const auto dot = [&](size_t m, size_t n) {
            return emitted(add(g, "MxDot", {param(g, element::u8, Shape{m, 16}), param(g, element::u8, Shape{m, 16}), param(g, element::u8, Shape{n, 16}),
                                            param(g, element::u8, Shape{n, 16})}));
        };
        const auto grouped = [&](size_t experts, size_t m, size_t rows, const char* act) {
            return emitted(add(g, "MxGroupedDot", {param(g, element::u8, Shape{m, 16}), param(g, element::u8, Shape{m, 16}), param(g, element::u8, Shape{experts, rows, 16}),
                                                   param(g, element::u8, Shape{experts, rows, 16}), param(g, element::i32, Shape{experts + 1})}, act));
        };
        EXPECT(choose(1 << 24, 4096, 32, false, 0, 256) != KERNELS && !dot(1 << 24, 4096).empty());
        EXPECT(choose(1 << 28, 4096, 32, false, 0, 256) == KERNELS && dot(1 << 28, 4096).empty());
        // experts of few rows each need a block of rows each
        const char* const gate = "{\"act\": \"silu_gate\"}";
        EXPECT(choose(1 << 14, 1 << 16, 32, true, 1 << 13, 256) != KERNELS && !grouped(1 << 13, 1 << 14, 1 << 17, gate).empty());
        EXPECT(choose(1 << 23, 1 << 16, 32, true, 1 << 23, 256) == KERNELS && grouped(1 << 23, 1 << 23, 1 << 17, gate).empty());
        EXPECT(choose(1 << 20, 4096, 32, false, 1 << 20, 256) == KERNELS && grouped(1 << 20, 1 << 20, 4096, "{}").empty());
    });
    return failures ? 1 : 0;
}
