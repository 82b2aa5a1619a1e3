// The operators on microscaled 4-bit numbers (MXFP4, include/nnf_hip_kernels.h), declared through the operator-plugin interface
// (REGISTER_OP / GenericOp, precedent: src/nnfusion/core/operators/generic_op/generic_op_define/MatMulAdd.cpp:6-35) like those
// of the integer formats (quant_ops.cpp).  A tensor of this format is two: codes u8 [.., rows, K/2] and scale bytes u8 [.., rows, S]
// with S = K/32 rounded up to 16.
//
//   MxQuantize    inputs: x f16 [rows, K] [, index i32 [n]] (attr has_index: row i of the results is x's row index[i])
//                 outputs: codes u8 [n, K/2], scales u8 [n, S]
//   MxDequantize  inputs: codes, scales                    output: f16 [rows, K]
//   MxDot         inputs: A codes [M, K/2], A scales, W codes [N, K/2], W scales [, bias f16 [N]] [, residual f16 [M, N]]
//                 attrs : has_bias false, has_residual false, act "none"|"silu_gate" (W: gate rows, then up rows)
//                 output: Y f16 [M, N]  (half of W's rows when act == "silu_gate")
//   MxGroupedDot  inputs: A codes [M, K/2], A scales, W codes [E, N, K/2], W scales [E, N, S], offsets i32 [E + 1]
//                 attrs : act;  output: Y f16 [M, N]; rows that belong to no group are not written
#include "../../nnf_mxfp4_plan.h"
#include "nnfusion/core/operators/generic_op/generic_op.hpp"

using namespace nnfusion;

namespace
{
    bool flag(std::shared_ptr<op::GenericOp> gop, const std::string& key) { return gop->localOpConfig.getRoot()[key].get<bool>(); }
    std::string text(std::shared_ptr<op::GenericOp> gop, const std::string& key) { return gop->localOpConfig.getRoot()[key].get<std::string>(); }

    // K of the pair (codes, scales) at inputs i, i + 1, whose leading axes agree
    size_t checked_pair(std::shared_ptr<op::GenericOp> gop, std::shared_ptr<graph::GNode> gnode, size_t i, size_t rank)
    {
        const Shape& c = gnode->get_input_shape(i);
        const Shape& s = gnode->get_input_shape(i + 1);
        OP_VALIDATION(gop, gnode->get_input_element_type(i) == element::u8 && gnode->get_input_element_type(i + 1) == element::u8)
            << "codes and scale bytes travel as u8";
        OP_VALIDATION(gop, c.size() == rank && s.size() == rank) << "bad ranks";
        const size_t K = 2 * c.back();
        OP_VALIDATION(gop, K <= (size_t)nnf::mx::MAX_K && nnf::mx::supported((int)K)) << "K must be a multiple of 32";
        OP_VALIDATION(gop, std::equal(c.begin(), c.end() - 1, s.begin()) && s.back() == (size_t)nnf::mx::scale_bytes((int)K))
            << "scales must be [.., K/32 rounded up to 16]";
        return K;
    }
    // columns of the product from the rows of a weight matrix
    size_t columns(std::shared_ptr<op::GenericOp> gop, size_t rows)
    {
        if (text(gop, "act") != "silu_gate")
            return rows;
        OP_VALIDATION(gop, rows % 2 == 0) << "gate|up weights need an even row count";
        return rows / 2;
    }
    bool known_act(const op::OpConfig::any& config)
    {
        const auto act = config.at("act").get<std::string>();
        return act == "none" || act == "silu_gate";
    }
} // namespace

REGISTER_OP(MxQuantize).attr<bool>("has_index", false).infershape([](std::shared_ptr<graph::GNode> gnode) -> void {
    auto gop = std::dynamic_pointer_cast<op::GenericOp>(gnode->get_op_ptr());
    NNFUSION_CHECK_NOT_NULLPTR(gop);
    const bool has_index = flag(gop, "has_index");
    OP_VALIDATION(gop, gnode->get_input_size() == (has_index ? 2u : 1u)) << "inputs: x [, index]";
    const Shape& x = gnode->get_input_shape(0);
    OP_VALIDATION(gop, x.size() == 2 && gnode->get_input_element_type(0) == element::f16) << "x must be f16 [rows, K]";
    OP_VALIDATION(gop, x[1] <= (size_t)nnf::mx::MAX_K && nnf::mx::supported((int)x[1])) << "K must be a multiple of 32";
    size_t rows = x[0];
    if (has_index)
    {
        const Shape& index = gnode->get_input_shape(1);
        OP_VALIDATION(gop, index.size() == 1 && gnode->get_input_element_type(1) == element::i32) << "index must be i32 [rows]";
        rows = index[0];
    }
    gnode->set_output_size(2);
    gnode->set_output_type_and_shape(0, element::u8, Shape{rows, x[1] / 2});
    gnode->set_output_type_and_shape(1, element::u8, Shape{rows, (size_t)nnf::mx::scale_bytes((int)x[1])});
});

REGISTER_OP(MxDequantize).infershape([](std::shared_ptr<graph::GNode> gnode) -> void {
    auto gop = std::dynamic_pointer_cast<op::GenericOp>(gnode->get_op_ptr());
    NNFUSION_CHECK_NOT_NULLPTR(gop);
    OP_VALIDATION(gop, gnode->get_input_size() == 2) << "inputs: codes, scales";
    const size_t K = checked_pair(gop, gnode, 0, 2);
    gnode->set_output_type_and_shape(0, element::f16, Shape{gnode->get_input_shape(0)[0], K});
});

REGISTER_OP(MxDot)
    .attr<bool>("has_bias", false)
    .attr<bool>("has_residual", false)
    .attr<std::string>("act", "none")
    .constrait(known_act)
    .infershape([](std::shared_ptr<graph::GNode> gnode) -> void {
        auto gop = std::dynamic_pointer_cast<op::GenericOp>(gnode->get_op_ptr());
        NNFUSION_CHECK_NOT_NULLPTR(gop);
        const bool bias = flag(gop, "has_bias"), residual = flag(gop, "has_residual");
        OP_VALIDATION(gop, gnode->get_input_size() == 4u + (bias ? 1 : 0) + (residual ? 1 : 0)) << "inputs: A, A scales, W, W scales [, bias] [, residual]";
        const size_t K = checked_pair(gop, gnode, 0, 2);
        OP_VALIDATION(gop, checked_pair(gop, gnode, 2, 2) == K) << "reduction axes do not match";
        const size_t M = gnode->get_input_shape(0)[0], N = columns(gop, gnode->get_input_shape(2)[0]);
        size_t i = 4;
        if (bias)
        {
            OP_VALIDATION(gop, gnode->get_input_element_type(i) == element::f16 && gnode->get_input_shape(i) == (Shape{N})) << "bias must be f16 [N]";
            ++i;
        }
        if (residual)
            OP_VALIDATION(gop, gnode->get_input_element_type(i) == element::f16 && gnode->get_input_shape(i) == (Shape{M, N})) << "residual must be f16 [M, N]";
        gnode->set_output_type_and_shape(0, element::f16, Shape{M, N});
    });

REGISTER_OP(MxGroupedDot).attr<std::string>("act", "none").constrait(known_act).infershape([](std::shared_ptr<graph::GNode> gnode) -> void {
    auto gop = std::dynamic_pointer_cast<op::GenericOp>(gnode->get_op_ptr());
    NNFUSION_CHECK_NOT_NULLPTR(gop);
    OP_VALIDATION(gop, gnode->get_input_size() == 5) << "inputs: A, A scales, W, W scales, offsets";
    const size_t K = checked_pair(gop, gnode, 0, 2);
    OP_VALIDATION(gop, checked_pair(gop, gnode, 2, 3) == K) << "reduction axes do not match";
    const Shape& w = gnode->get_input_shape(2);
    OP_VALIDATION(gop, gnode->get_input_element_type(4) == element::i32 && gnode->get_input_shape(4) == (Shape{w[0] + 1})) << "offsets must be i32 [experts + 1]";
    gnode->set_output_type_and_shape(0, element::f16, Shape{gnode->get_input_shape(0)[0], columns(gop, w[1])});
});
