// nnf_compile_example: builds a small graph around the quantized operators, runs the ROCm engine
// (device dispatch -> kernel selection -> HIP code generation) and leaves the generated project in
// <out_dir>.  It stands where the reference's `nnfusion` CLI stands (src/tools/nnfusion/nnfusion.cpp:57-188)
// for the one path this build covers; model import (ONNX / TensorFlow frontends) is not part of it.
// Constants come from the seeded generator (seed 0, the stream ids of nnfusion_amd/datagen.py), so a
// caller can regenerate the same weights to check the result.
//
//   nnf_compile_example quant_dot <out_dir> M N K
//   nnf_compile_example w8a8      <out_dir> M N K
//   nnf_compile_example mlp       <out_dir> M H I       (one FusedQuantMLP node)
//   nnf_compile_example mlp_nodes <out_dir> M H I       (two QuantDot nodes: rms+gate|up, down+residual)
//   nnf_compile_example mlp_graph <out_dir> M H I       (the unfused block: RMSNorm, gate / up / down QuantDots,
//                                                         Swish, Multiply, Add; the fusion pass folds it into one node)
//   nnf_compile_example qkv_graph <out_dir> M N K       (RMSNorm feeding three QuantDots of N rows each; merged
//                                                         into one 3N-row QuantDot + three Slices; three results)
//   nnf_compile_example mx_experts <out_dir> M H I       (a mixture of four experts on MXFP4: rows picked by an index are quantised,
//                                                         gate | up with SiLU-gate, quantised, down; x, index, offsets are inputs)
//   nnf_compile_example fp8_experts <out_dir> M H I      (a mixture of eight experts in block-scaled 8-bit floating point: three of them
//                                                         for each token by its logits and a bias, gate | up with SiLU-gate, down, weighted back onto x; x, logits, bias are inputs)
// every form: [include_dir lib_dir [kernel_profiling_dir [prepare]]] at the end; a kernel_profiling_dir switches
// profiling-based kernel selection on (every candidate kernel of a QuantDot node is timed on the GPU)
//   nnf_compile_example onnx      <out_dir> <model.onnx> [include_dir lib_dir]
//                                                        (an ONNX model of the quantized path: MatMulNBits,
//                                                         SimplifiedLayerNormalization, Sigmoid, Mul, Add)
#include "../../nnf_mxfp4_plan.h"
#include "../nnf_datagen.h"
#include "nnfusion/core/operators/generic_op/generic_op.hpp"
#include "nnfusion/engine/pass/codegen/base_codegen_pass.hpp"
#include "nnfusion/frontend/onnx_import/onnx.hpp"

#include <cstdlib>
#include <cstring>

using namespace nnfusion;

namespace
{
    // stream ids shared with nnfusion_amd/datagen.py
    enum
    {
        S_ACT = 1, S_WQ, S_SCALE, S_GAMMA, S_A8, S_W8, S_STOK, S_SCH, S_WQ2, S_SCALE2, S_BIAS, S_RES, S_ZP, S_MXS, S_MXS2
    };

    std::shared_ptr<graph::GNode> constant_u4(graph::Graph& g, uint64_t stream, size_t n, size_t k)
    {
        std::vector<uint8_t> data(n * k / 2);
        nnf_gen_uniform_u4_packed(0, stream, data.data(), n * k);
        return g.add_node_and_edge(std::make_shared<op::Constant>(element::u8, Shape{n, k / 2}, data.data()), graph::GNodeVector{});
    }
    std::shared_ptr<graph::GNode> constant_scales(graph::Graph& g, uint64_t stream, size_t n, size_t groups)
    {
        std::vector<uint16_t> data(n * groups);
        nnf_gen_uniform_f16(0, stream, 0.005, 0.02, data.data(), data.size());
        return g.add_node_and_edge(std::make_shared<op::Constant>(element::f16, Shape{n, groups}, data.data()), graph::GNodeVector{});
    }
    // the codes and scale bytes (2^-9 .. 2^-3) of `experts` matrices
    std::pair<std::shared_ptr<graph::GNode>, std::shared_ptr<graph::GNode>> constant_mx(graph::Graph& g, uint64_t codes, uint64_t scales, size_t experts,
                                                                                        size_t n, size_t k)
    {
        std::vector<uint8_t> data(experts * n * k / 2);
        nnf_gen_uniform_u4_packed(0, codes, data.data(), experts * n * k);
        const size_t stride = (size_t)nnf::mx::scale_bytes((int)k);
        std::vector<int8_t> bytes(experts * n * stride);
        nnf_gen_uniform_i8(0, scales, 118, 124, bytes.data(), bytes.size());
        return {g.add_node_and_edge(std::make_shared<op::Constant>(element::u8, Shape{experts, n, k / 2}, data.data()), graph::GNodeVector{}),
                g.add_node_and_edge(std::make_shared<op::Constant>(element::u8, Shape{experts, n, stride}, bytes.data()), graph::GNodeVector{})};
    }
    // codes (either sign, up to 0x6F: 240) and scales of `experts` weight matrices of parts * n rows
    std::pair<std::shared_ptr<graph::GNode>, std::shared_ptr<graph::GNode>> constant_fp8(graph::Graph& g, uint64_t codes, uint64_t scales, size_t experts,
                                                                                         size_t parts, size_t n, size_t k)
    {
        std::vector<int8_t> data(experts * parts * n * k);
        nnf_gen_uniform_i8(0, codes, -111, 111, data.data(), data.size());
        for (auto& v : data)
            v = (int8_t)(v < 0 ? 0x80 | -v : v);
        const size_t nb = parts * ((n + 127) / 128), kb = (k + 127) / 128;
        std::vector<float> s(experts * nb * kb);
        nnf_gen_uniform_f32(0, scales, 0.0005, 0.002, s.data(), s.size());
        return {g.add_node_and_edge(std::make_shared<op::Constant>(element::u8, Shape{experts, parts * n, k}, data.data()), graph::GNodeVector{}),
                g.add_node_and_edge(std::make_shared<op::Constant>(element::f32, Shape{experts, nb, kb}, s.data()), graph::GNodeVector{})};
    }
} // namespace

int main(int argc, char** argv)
{
    const bool from_onnx = argc >= 4 && std::string(argv[1]) == "onnx";
    if (argc < 6 && !(from_onnx && argc >= 4))
    {
        fprintf(stderr, "usage: %s <quant_dot|w8a8|mlp|mlp_nodes|mlp_graph|qkv_graph|mx_experts|fp8_experts> <out_dir> <d0> <d1> <d2> [include_dir lib_dir]\n"
                        "       %s onnx <out_dir> <model.onnx> [include_dir lib_dir]\n", argv[0], argv[0]);
        return 2;
    }
    const std::string kind = argv[1], out_dir = argv[2];
    const size_t d0 = from_onnx ? 0 : strtoul(argv[3], nullptr, 10), d1 = from_onnx ? 0 : strtoul(argv[4], nullptr, 10),
                 d2 = from_onnx ? 0 : strtoul(argv[5], nullptr, 10);
    const int dirs_at = from_onnx ? 4 : 6; // where the optional include / library directories start
    auto g = std::make_shared<graph::Graph>();
    try
    {
        if (from_onnx)
            g = frontend::load_onnx_model(argv[3]);
        else
        if (kind == "quant_dot")
        {
            const size_t M = d0, N = d1, K = d2;
            auto a = g->add_node_and_edge(std::make_shared<op::Parameter>(element::f16, Shape{M, K}), graph::GNodeVector{});
            auto wq = constant_u4(*g, S_WQ, N, K);
            auto s = constant_scales(*g, S_SCALE, N, K / 128);
            auto dot = g->add_node_and_edge(std::make_shared<op::GenericOp>("linear", "QuantDot", op::OpConfig::any()), {a, wq, s});
            g->add_node_and_edge(std::make_shared<op::Result>(), {dot});
        }
        else if (kind == "w8a8")
        {
            const size_t M = d0, N = d1, K = d2;
            auto a = g->add_node_and_edge(std::make_shared<op::Parameter>(element::i8, Shape{M, K}), graph::GNodeVector{});
            auto st = g->add_node_and_edge(std::make_shared<op::Parameter>(element::f32, Shape{M}), graph::GNodeVector{});
            std::vector<int8_t> w(N * K);
            nnf_gen_uniform_i8(0, S_W8, -127, 127, w.data(), w.size());
            std::vector<float> sch(N);
            nnf_gen_uniform_f32(0, S_SCH, 0.001, 0.01, sch.data(), sch.size());
            auto wn = g->add_node_and_edge(std::make_shared<op::Constant>(element::i8, Shape{N, K}, w.data()), graph::GNodeVector{});
            auto sn = g->add_node_and_edge(std::make_shared<op::Constant>(element::f32, Shape{N}, sch.data()), graph::GNodeVector{});
            auto dot = g->add_node_and_edge(std::make_shared<op::GenericOp>("linear_w8a8", "QuantDotW8A8", op::OpConfig::any()),
                                            {a, st, wn, sn});
            g->add_node_and_edge(std::make_shared<op::Result>(), {dot});
        }
        else if (kind == "mlp" || kind == "mlp_nodes")
        {
            const size_t M = d0, H = d1, I = d2;
            auto x = g->add_node_and_edge(std::make_shared<op::Parameter>(element::f16, Shape{M, H}), graph::GNodeVector{});
            std::vector<uint16_t> gam(H);
            nnf_gen_normal_f16(0, S_GAMMA, 1.0, 0.1, gam.data(), H);
            auto gamma = g->add_node_and_edge(std::make_shared<op::Constant>(element::f16, Shape{H}, gam.data()), graph::GNodeVector{});
            auto wgu = constant_u4(*g, S_WQ, 2 * I, H);
            auto sgu = constant_scales(*g, S_SCALE, 2 * I, H / 128);
            auto wd = constant_u4(*g, S_WQ2, H, I);
            auto sd = constant_scales(*g, S_SCALE2, H, I / 128);
            std::shared_ptr<graph::GNode> out;
            if (kind == "mlp")
            {
                out = g->add_node_and_edge(std::make_shared<op::GenericOp>("mlp", "FusedQuantMLP", op::OpConfig::any()),
                                           {x, gamma, wgu, sgu, wd, sd});
            }
            else
            {
                auto gate_up = g->add_node_and_edge(
                    std::make_shared<op::GenericOp>("gate_up", "QuantDot",
                                                    op::OpConfig::any::parse("{\"rms_norm\": true, \"act\": \"silu_gate\"}")),
                    {x, wgu, sgu, gamma});
                out = g->add_node_and_edge(
                    std::make_shared<op::GenericOp>("down", "QuantDot", op::OpConfig::any::parse("{\"has_residual\": true}")),
                    {gate_up, wd, sd, x});
            }
            g->add_node_and_edge(std::make_shared<op::Result>(), {out});
        }
        else if (kind == "mlp_graph")
        {
            const size_t M = d0, H = d1, I = d2;
            auto x = g->add_node_and_edge(std::make_shared<op::Parameter>(element::f16, Shape{M, H}), graph::GNodeVector{});
            std::vector<uint16_t> gam(H);
            nnf_gen_normal_f16(0, S_GAMMA, 1.0, 0.1, gam.data(), H);
            auto gamma = g->add_node_and_edge(std::make_shared<op::Constant>(element::f16, Shape{H}, gam.data()), graph::GNodeVector{});
            // the same [gate; up] bytes as the other MLP kinds, cut into the two projections
            std::vector<uint8_t> wgu(2 * I * H / 2);
            nnf_gen_uniform_u4_packed(0, S_WQ, wgu.data(), 2 * I * H);
            std::vector<uint16_t> sgu(2 * I * (H / 128));
            nnf_gen_uniform_f16(0, S_SCALE, 0.005, 0.02, sgu.data(), sgu.size());
            auto cst = [&](const element::Type& t, const Shape& s, const void* p) {
                return g->add_node_and_edge(std::make_shared<op::Constant>(t, s, p), graph::GNodeVector{});
            };
            auto wg = cst(element::u8, Shape{I, H / 2}, wgu.data());
            auto wu = cst(element::u8, Shape{I, H / 2}, wgu.data() + I * H / 2);
            auto sg = cst(element::f16, Shape{I, H / 128}, sgu.data());
            auto su = cst(element::f16, Shape{I, H / 128}, sgu.data() + I * (H / 128));
            auto wd = constant_u4(*g, S_WQ2, H, I);
            auto sd = constant_scales(*g, S_SCALE2, H, I / 128);
            auto any = op::OpConfig::any();
            auto n = g->add_node_and_edge(std::make_shared<op::GenericOp>("norm", "RMSNorm", any), {x, gamma});
            auto gate = g->add_node_and_edge(std::make_shared<op::GenericOp>("gate", "QuantDot", any), {n, wg, sg});
            auto up = g->add_node_and_edge(std::make_shared<op::GenericOp>("up", "QuantDot", any), {n, wu, su});
            auto act = g->add_node_and_edge(std::make_shared<op::GenericOp>("act", "Swish", any), {gate});
            auto h = g->add_node_and_edge(std::make_shared<op::GenericOp>("h", "Multiply", any), {act, up});
            auto down = g->add_node_and_edge(std::make_shared<op::GenericOp>("down", "QuantDot", any), {h, wd, sd});
            auto out = g->add_node_and_edge(std::make_shared<op::GenericOp>("out", "Add", any), {x, down});
            g->add_node_and_edge(std::make_shared<op::Result>(), {out});
        }
        else if (kind == "mx_experts")
        {
            const size_t M = d0, H = d1, I = d2, E = 4;
            auto x = g->add_node_and_edge(std::make_shared<op::Parameter>(element::f16, Shape{M, H}), graph::GNodeVector{});
            auto index = g->add_node_and_edge(std::make_shared<op::Parameter>(element::i32, Shape{2 * M}), graph::GNodeVector{});
            auto offsets = g->add_node_and_edge(std::make_shared<op::Parameter>(element::i32, Shape{E + 1}), graph::GNodeVector{});
            auto up = constant_mx(*g, S_WQ, S_MXS, E, 2 * I, H), down = constant_mx(*g, S_WQ2, S_MXS2, E, H, I);
            using Inputs = std::vector<std::pair<std::shared_ptr<graph::GNode>, int>>;
            auto a = g->add_node_and_edge(std::make_shared<op::GenericOp>("quantize", "MxQuantize", op::OpConfig::any::parse("{\"has_index\": true}")),
                                          Inputs{{x, 0}, {index, 0}});
            auto h = g->add_node_and_edge(std::make_shared<op::GenericOp>("gate_up", "MxGroupedDot", op::OpConfig::any::parse("{\"act\": \"silu_gate\"}")),
                                          Inputs{{a, 0}, {a, 1}, {up.first, 0}, {up.second, 0}, {offsets, 0}});
            auto b = g->add_node_and_edge(std::make_shared<op::GenericOp>("quantize_h", "MxQuantize", op::OpConfig::any()), Inputs{{h, 0}});
            auto y = g->add_node_and_edge(std::make_shared<op::GenericOp>("down", "MxGroupedDot", op::OpConfig::any()),
                                          Inputs{{b, 0}, {b, 1}, {down.first, 0}, {down.second, 0}, {offsets, 0}});
            g->add_node_and_edge(std::make_shared<op::Result>(), {y});
        }
        else if (kind == "fp8_experts")
        {
            const size_t M = d0, H = d1, I = d2, E = 8;
            auto x = g->add_node_and_edge(std::make_shared<op::Parameter>(element::f16, Shape{M, H}), graph::GNodeVector{});
            auto logits = g->add_node_and_edge(std::make_shared<op::Parameter>(element::f32, Shape{M, E}), graph::GNodeVector{});
            auto bias = g->add_node_and_edge(std::make_shared<op::Parameter>(element::f32, Shape{E}), graph::GNodeVector{});
            auto up = constant_fp8(*g, S_WQ, S_MXS, E, 2, I, H), down = constant_fp8(*g, S_WQ2, S_MXS2, E, 1, H, I);
            using Inputs = std::vector<std::pair<std::shared_ptr<graph::GNode>, int>>;
            const auto node = [&](const char* name, const char* type, const char* config, const Inputs& in) {
                return g->add_node_and_edge(std::make_shared<op::GenericOp>(name, type, op::OpConfig::any::parse(config)), in);
            };
            auto to = node("route", "MoeRoute", "{\"has_bias\": true, \"k\": 3, \"score\": \"sigmoid\", \"groups\": 4, \"top_groups\": 2, \"group_top\": 2, \"scale\": 2.5}",
                           Inputs{{logits, 0}, {bias, 0}});
            auto a = node("quantize", "Fp8Quantize", "{\"has_index\": true}", Inputs{{x, 0}, {to, 2}});
            auto h = node("gate_up", "Fp8GroupedDot", "{\"act\": \"silu_gate\"}", Inputs{{a, 0}, {a, 1}, {up.first, 0}, {up.second, 0}, {to, 3}});
            auto b = node("quantize_h", "Fp8Quantize", "{}", Inputs{{h, 0}});
            auto y = node("down", "Fp8GroupedDot", "{}", Inputs{{b, 0}, {b, 1}, {down.first, 0}, {down.second, 0}, {to, 3}});
            auto out = node("combine", "MoeCombine", "{\"has_residual\": true}", Inputs{{y, 0}, {to, 0}, {to, 4}, {x, 0}});
            g->add_node_and_edge(std::make_shared<op::Result>(), {out});
        }
        else if (kind == "qkv_graph")
        {
            const size_t M = d0, N = d1, K = d2;
            auto x = g->add_node_and_edge(std::make_shared<op::Parameter>(element::f16, Shape{M, K}), graph::GNodeVector{});
            std::vector<uint16_t> gam(K);
            nnf_gen_normal_f16(0, S_GAMMA, 1.0, 0.1, gam.data(), K);
            auto gamma = g->add_node_and_edge(std::make_shared<op::Constant>(element::f16, Shape{K}, gam.data()), graph::GNodeVector{});
            // one [3N, K] weight block (the bytes of quant_dot with N' = 3N), cut into q, k and v
            std::vector<uint8_t> w(3 * N * K / 2);
            nnf_gen_uniform_u4_packed(0, S_WQ, w.data(), 3 * N * K);
            std::vector<uint16_t> sc(3 * N * (K / 128));
            nnf_gen_uniform_f16(0, S_SCALE, 0.005, 0.02, sc.data(), sc.size());
            auto any = op::OpConfig::any();
            auto n = g->add_node_and_edge(std::make_shared<op::GenericOp>("norm", "RMSNorm", any), {x, gamma});
            const char* names[3] = {"q_proj", "k_proj", "v_proj"};
            for (int i = 0; i < 3; ++i)
            {
                auto wq = g->add_node_and_edge(std::make_shared<op::Constant>(element::u8, Shape{N, K / 2}, w.data() + i * N * K / 2),
                                               graph::GNodeVector{});
                auto s = g->add_node_and_edge(
                    std::make_shared<op::Constant>(element::f16, Shape{N, K / 128}, sc.data() + i * N * (K / 128)),
                    graph::GNodeVector{});
                auto dot = g->add_node_and_edge(std::make_shared<op::GenericOp>(names[i], "QuantDot", any), {n, wq, s});
                g->add_node_and_edge(std::make_shared<op::Result>(), {dot});
            }
        }
        else
        {
            fprintf(stderr, "unknown kind %s\n", kind.c_str());
            return 2;
        }
        ROCmEngine engine(out_dir);
        engine.quant_gemm_fusion = kind == "qkv_graph";
        if (argc >= dirs_at + 2)
        {
            engine.pass.kernels_include_dir = argv[dirs_at];
            engine.pass.kernels_lib_dir = argv[dirs_at + 1];
        }
        // [kernel_profiling_dir [prepare]]: profiling-based kernel selection (-fkernel_selection of the reference);
        // "prepare" only builds the single-kernel harnesses, for a later run on a host with the GPU
        if (argc >= dirs_at + 3)
        {
            engine.kernel_selection = true;
            nnfusion::min_log_level() = 1; // the time of every candidate is logged at INFO
            engine.kernel_profiling_dir = argv[dirs_at + 2];
            engine.kernel_profiling_runs = 50;
            engine.kernel_selection_prepare_only = argc >= dirs_at + 4 && std::string(argv[dirs_at + 3]) == "prepare";
        }
        engine.pass.exit_after_codegen = false;
        engine.run_on_graph(g);
    }
    catch (const std::exception& e)
    {
        fprintf(stderr, "nnf_compile_example: %s\n", e.what());
        return 1;
    }
    if (argc >= dirs_at + 4 && std::string(argv[dirs_at + 3]) == "prepare")
        printf("kernel-selection harnesses of %s built in %s\n", kind.c_str(), argv[dirs_at + 2]);
    else
        printf("generated %s in %s\n", kind.c_str(), out_dir.c_str());
    return 0;
}
