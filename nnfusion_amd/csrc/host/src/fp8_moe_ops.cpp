// The operators around a mixture's experts and their products in block-scaled 8-bit floating point (include/nnf_hip_kernels.h), declared
// through the operator-plugin interface (REGISTER_OP / GenericOp, precedent:
// src/nnfusion/core/operators/generic_op/generic_op_define/MatMulAdd.cpp:6-35) like those on MXFP4 (mxfp4_ops.cpp).  Codes travel as u8.
//
//   MoeRoute      inputs: logits f32 | f16 [tokens, E] [, bias f32 [E]] [, tokens i32 [1]]
//                 attrs : has_bias, has_tokens, k, score "softmax"|"sigmoid", groups, top_groups, group_top, renormalize, scale
//                 outputs: weights f32 [tokens, k], experts i32 [tokens, k], rows i32 [tokens k], offsets i32 [E + 1], positions i32 [tokens, k]
//   MoeCombine    inputs: x f16 [rows, N], weights f32 [tokens, k], positions i32 [tokens, k] [, residual f16 [tokens, N]] (attr has_residual)
//                 output: f16 [tokens, N]
//   Fp8Quantize   inputs: x f16 [rows, K] [, index i32 [n]] (attr has_index)
//                 outputs: codes u8 [n, K], scales f32 [ceil(K/128), n]
//   Fp8Dot        inputs: A codes [M, K], A scales, W codes [N, K], W scales f32 [ceil(N/128), ceil(K/128)] [, bias f16 [N]] [, residual f16 [M, N]]
//                 attrs : has_bias false, has_residual false, act "none"|"silu_gate" (W: gate rows, then up rows, each with blocks of their own)
//                 output: f16 [M, N]
//   Fp8GroupedDot inputs: A codes, A scales, W codes [E, N, K], W scales [E, .., ..], offsets i32 [E + 1]
//                 attrs : act;  output: f16 [M, N]; rows that belong to no group are not written
#include "../../nnf_fp8_plan.h"
#include "../../nnf_moe_plan.h"
#include "nnfusion/core/operators/generic_op/generic_op.hpp"

using namespace nnfusion;

namespace
{
    using Gop = std::shared_ptr<op::GenericOp>;
    using Node = std::shared_ptr<graph::GNode>;

    Gop generic(const Node& gnode)
    {
        auto gop = std::dynamic_pointer_cast<op::GenericOp>(gnode->get_op_ptr());
        NNFUSION_CHECK_NOT_NULLPTR(gop);
        return gop;
    }
    bool flag(const Gop& gop, const std::string& key) { return gop->localOpConfig.getRoot()[key].get<bool>(); }
    int number(const Gop& gop, const std::string& key) { return gop->localOpConfig.getRoot()[key].get<int>(); }
    bool is(const Node& gnode, size_t i, const element::Type& type, const Shape& shape)
    {
        return gnode->get_input_element_type(i) == type && gnode->get_input_shape(i) == shape;
    }
    size_t blocks(size_t n) { return (n + nnf::fp8::BLOCK - 1) / nnf::fp8::BLOCK; }

    // K of codes [.., K] at input i
    size_t checked_codes(const Gop& gop, const Node& gnode, size_t i, size_t rank)
    {
        const Shape& c = gnode->get_input_shape(i);
        OP_VALIDATION(gop, gnode->get_input_element_type(i) == element::u8 && c.size() == rank) << "codes travel as u8, of " << rank << " axes";
        OP_VALIDATION(gop, c.back() <= (size_t)nnf::fp8::MAX_K && nnf::fp8::supported((int)c.back())) << "K must be a multiple of 16";
        return c.back();
    }
    // columns of the product from the rows of a weight matrix
    size_t columns(const Gop& gop, size_t rows)
    {
        if (gop->localOpConfig.getRoot()["act"].get<std::string>() != "silu_gate")
            return rows;
        OP_VALIDATION(gop, rows % 2 == 0) << "gate|up weights need an even row count";
        return rows / 2;
    }
    // the operands at inputs 0 .. 3, of one weight matrix (rank 2) or several (3) -> M, N
    std::pair<size_t, size_t> checked_product(const Gop& gop, const Node& gnode, size_t rank)
    {
        const size_t K = checked_codes(gop, gnode, 0, 2), M = gnode->get_input_shape(0)[0];
        OP_VALIDATION(gop, checked_codes(gop, gnode, 2, rank) == K) << "reduction axes do not match";
        OP_VALIDATION(gop, is(gnode, 1, element::f32, Shape{blocks(K), M})) << "scales of A must be f32 [ceil(K/128), M]";
        Shape w = gnode->get_input_shape(2);
        const size_t rows = w[rank - 2], N = columns(gop, rows);
        w[rank - 2] = rows / (N ? N : 1) * blocks(N), w[rank - 1] = blocks(K);
        OP_VALIDATION(gop, is(gnode, 3, element::f32, w)) << "scales of W must be f32 [.., ceil(N/128), ceil(K/128)], with silu_gate twice the blocks of N";
        return {M, N};
    }
    bool known_act(const op::OpConfig::any& config)
    {
        const auto act = config.at("act").get<std::string>();
        return act == "none" || act == "silu_gate";
    }
    bool known_score(const op::OpConfig::any& config)
    {
        const auto score = config.at("score").get<std::string>();
        return score == "softmax" || score == "sigmoid";
    }
} // namespace

REGISTER_OP(MoeRoute)
    .attr<bool>("has_bias", false)
    .attr<bool>("has_tokens", false)
    .attr<int>("k", 1)
    .attr<std::string>("score", "softmax")
    .attr<int>("groups", 1)
    .attr<int>("top_groups", 1)
    .attr<int>("group_top", 1)
    .attr<bool>("renormalize", true)
    .attr<double>("scale", 1.0)
    .constrait(known_score)
    .infershape([](Node gnode) -> void {
        auto gop = generic(gnode);
        const bool bias = flag(gop, "has_bias"), tokens = flag(gop, "has_tokens");
        OP_VALIDATION(gop, gnode->get_input_size() == 1u + (bias ? 1 : 0) + (tokens ? 1 : 0)) << "inputs: logits [, bias] [, tokens]";
        const Shape& l = gnode->get_input_shape(0);
        OP_VALIDATION(gop, l.size() == 2 && (gnode->get_input_element_type(0) == element::f32 || gnode->get_input_element_type(0) == element::f16))
            << "logits must be f32 or f16 [tokens, experts]";
        const size_t T = l[0], E = l[1];
        OP_VALIDATION(gop, E <= (size_t)nnf::moe::MAX_EXPERTS &&
                               nnf::moe::choosable((int)E, number(gop, "k"), number(gop, "groups"), number(gop, "top_groups"), number(gop, "group_top")))
            << "k experts cannot be chosen among these groups";
        OP_VALIDATION(gop, !bias || is(gnode, 1, element::f32, Shape{E})) << "bias must be f32 [experts]";
        OP_VALIDATION(gop, !tokens || is(gnode, bias ? 2 : 1, element::i32, Shape{1})) << "tokens must be i32 [1]";
        const size_t k = (size_t)number(gop, "k");
        gnode->set_output_size(5);
        gnode->set_output_type_and_shape(0, element::f32, Shape{T, k});
        gnode->set_output_type_and_shape(1, element::i32, Shape{T, k});
        gnode->set_output_type_and_shape(2, element::i32, Shape{T * k});
        gnode->set_output_type_and_shape(3, element::i32, Shape{E + 1});
        gnode->set_output_type_and_shape(4, element::i32, Shape{T, k});
    });

REGISTER_OP(MoeCombine).attr<bool>("has_residual", false).infershape([](Node gnode) -> void {
    auto gop = generic(gnode);
    const bool residual = flag(gop, "has_residual");
    OP_VALIDATION(gop, gnode->get_input_size() == 3u + (residual ? 1 : 0)) << "inputs: x, weights, positions [, residual]";
    const Shape &x = gnode->get_input_shape(0), &w = gnode->get_input_shape(1);
    OP_VALIDATION(gop, x.size() == 2 && gnode->get_input_element_type(0) == element::f16) << "x must be f16 [rows, N]";
    OP_VALIDATION(gop, w.size() == 2 && gnode->get_input_element_type(1) == element::f32) << "weights must be f32 [tokens, k]";
    OP_VALIDATION(gop, is(gnode, 2, element::i32, w)) << "positions must be i32 [tokens, k]";
    const Shape y{w[0], x[1]};
    OP_VALIDATION(gop, !residual || is(gnode, 3, element::f16, y)) << "residual must be f16 [tokens, N]";
    gnode->set_output_type_and_shape(0, element::f16, y);
});

REGISTER_OP(Fp8Quantize).attr<bool>("has_index", false).infershape([](Node gnode) -> void {
    auto gop = generic(gnode);
    const bool has_index = flag(gop, "has_index");
    OP_VALIDATION(gop, gnode->get_input_size() == (has_index ? 2u : 1u)) << "inputs: x [, index]";
    const Shape& x = gnode->get_input_shape(0);
    OP_VALIDATION(gop, x.size() == 2 && gnode->get_input_element_type(0) == element::f16) << "x must be f16 [rows, K]";
    OP_VALIDATION(gop, x[1] <= (size_t)nnf::fp8::MAX_K && nnf::fp8::supported((int)x[1])) << "K must be a multiple of 16";
    size_t rows = x[0];
    if (has_index)
    {
        const Shape& index = gnode->get_input_shape(1);
        OP_VALIDATION(gop, index.size() == 1 && gnode->get_input_element_type(1) == element::i32) << "index must be i32 [rows]";
        rows = index[0];
    }
    gnode->set_output_size(2);
    gnode->set_output_type_and_shape(0, element::u8, Shape{rows, x[1]});
    gnode->set_output_type_and_shape(1, element::f32, Shape{blocks(x[1]), rows});
});

REGISTER_OP(Fp8Dot)
    .attr<bool>("has_bias", false)
    .attr<bool>("has_residual", false)
    .attr<std::string>("act", "none")
    .constrait(known_act)
    .infershape([](Node gnode) -> void {
        auto gop = generic(gnode);
        const bool bias = flag(gop, "has_bias"), residual = flag(gop, "has_residual");
        OP_VALIDATION(gop, gnode->get_input_size() == 4u + (bias ? 1 : 0) + (residual ? 1 : 0)) << "inputs: A, A scales, W, W scales [, bias] [, residual]";
        const auto size = checked_product(gop, gnode, 2);
        const Shape y{size.first, size.second};
        OP_VALIDATION(gop, !bias || is(gnode, 4, element::f16, Shape{y[1]})) << "bias must be f16 [N]";
        OP_VALIDATION(gop, !residual || is(gnode, bias ? 5 : 4, element::f16, y)) << "residual must be f16 [M, N]";
        gnode->set_output_type_and_shape(0, element::f16, y);
    });

REGISTER_OP(Fp8GroupedDot).attr<std::string>("act", "none").constrait(known_act).infershape([](Node gnode) -> void {
    auto gop = generic(gnode);
    OP_VALIDATION(gop, gnode->get_input_size() == 5) << "inputs: A, A scales, W, W scales, offsets";
    const auto size = checked_product(gop, gnode, 3);
    OP_VALIDATION(gop, is(gnode, 4, element::i32, Shape{gnode->get_input_shape(2)[0] + 1})) << "offsets must be i32 [experts + 1]";
    gnode->set_output_type_and_shape(0, element::f16, Shape{size.first, size.second});
});
