// Kernel emitters of the operators on microscaled 4-bit numbers (mxfp4_ops.cpp) for ROCM_GPU: each emits a host function around one
// call into the launcher library, like the emitters of the integer formats (quant_emitters.cpp).
#include "../../nnf_mxfp4_plan.h"
#include "nnf_hip_kernels.h"
#include "nnfusion/core/kernels/hip_gpu/hip_emitter.hpp"
#include "nnfusion/core/kernels/kernel_registration.hpp"
#include "nnfusion/core/operators/generic_op/generic_op.hpp"

#include <climits>

namespace nnfusion
{
    namespace kernels
    {
        namespace hip
        {
            namespace mx = nnf::mx;

            class MxEmitter : public HipLibEmitter
            {
            public:
                using HipLibEmitter::HipLibEmitter;

            protected:
                std::shared_ptr<op::GenericOp> generic() const { return std::dynamic_pointer_cast<op::GenericOp>(m_context->op); }
                const Shape& input(size_t i) const { return m_context->inputs[i]->get_shape(); }
                // every tensor has elements, and sizes that the calls' ints hold
                bool sized() const
                {
                    for (auto* list : {&m_context->inputs, &m_context->outputs})
                        for (auto& t : *list)
                            for (size_t n : t->get_shape())
                                if (n == 0 || n > (size_t)INT_MAX)
                                    return false;
                    return true;
                }
                static const char* act_enum(bool gate) { return gate ? "NNF_ACT_SILU_GATE" : "NNF_ACT_NONE"; }
                LanguageUnit_p call(const std::string& name, const std::string& arguments)
                {
                    LanguageUnit_p lu(new LanguageUnit(get_function_name()));
                    *lu << "NNF_HIP_CHECK(" << name << "(stream, " << arguments << "));\n";
                    return lu;
                }
            };

            class MxQuantize : public MxEmitter
            {
            public:
                explicit MxQuantize(std::shared_ptr<KernelContext> ctx)
                    : MxEmitter(ctx)
                {
                }
                LanguageUnit_p emit_function_body() override
                {
                    auto gop = generic();
                    if (!gop || !sized())
                        return nullptr;
                    if (!mx::convertible((int)m_context->outputs[0]->get_shape()[0], (int)input(0)[1]))
                        return nullptr;
                    const bool has_index = gop->localOpConfig.getRoot()["has_index"].get<bool>();
                    std::ostringstream ss;
                    ss << "input0, " << (has_index ? "input1" : "nullptr") << ", output0, output1, " << m_context->outputs[0]->get_shape()[0] << ", "
                       << input(0)[0] << ", " << input(0)[1];
                    return call("nnf_mxfp4_quantize_f16", ss.str());
                }
            };

            class MxDequantize : public MxEmitter
            {
            public:
                explicit MxDequantize(std::shared_ptr<KernelContext> ctx)
                    : MxEmitter(ctx)
                {
                }
                LanguageUnit_p emit_function_body() override
                {
                    if (!generic() || !sized() || !mx::convertible((int)input(0)[0], 2 * (int)input(0)[1]))
                        return nullptr;
                    std::ostringstream ss;
                    ss << "input0, input1, output0, " << input(0)[0] << ", " << 2 * input(0)[1];
                    return call("nnf_mxfp4_dequantize_f16", ss.str());
                }
            };

            class MxDot : public MxEmitter
            {
            public:
                explicit MxDot(std::shared_ptr<KernelContext> ctx)
                    : MxEmitter(ctx)
                {
                }
                LanguageUnit_p emit_function_body() override
                {
                    auto gop = generic();
                    if (!gop || !sized())
                        return nullptr;
                    auto& cfg = gop->localOpConfig.getRoot();
                    const bool bias = cfg["has_bias"].get<bool>(), residual = cfg["has_residual"].get<bool>();
                    const bool gate = cfg["act"].get<std::string>() == "silu_gate";
                    const Shape& y = m_context->outputs[0]->get_shape();
                    // what the launcher declines
                    if ((gate && (bias || residual)) || !mx::servable((int)y[0], (int)y[1], 2 * (int)input(0)[1], gate, 0))
                        return nullptr;
                    std::ostringstream ss;
                    ss << "input0, input1, input2, input3, output0, " << y[0] << ", " << y[1] << ", " << 2 * input(0)[1] << ", "
                       << (bias ? "input4" : "nullptr") << ", " << (residual ? (bias ? "input5" : "input4") : "nullptr") << ", " << act_enum(gate)
                       << ", nullptr, 0";
                    return call("nnf_mxfp4_gemm", ss.str());
                }
            };

            class MxGroupedDot : public MxEmitter
            {
            public:
                explicit MxGroupedDot(std::shared_ptr<KernelContext> ctx)
                    : MxEmitter(ctx)
                {
                }
                LanguageUnit_p emit_function_body() override
                {
                    auto gop = generic();
                    if (!gop || !sized())
                        return nullptr;
                    const bool gate = gop->localOpConfig.getRoot()["act"].get<std::string>() == "silu_gate";
                    const Shape& y = m_context->outputs[0]->get_shape();
                    if (!mx::servable((int)y[0], (int)y[1], 2 * (int)input(0)[1], gate, (int)input(2)[0]))
                        return nullptr;
                    std::ostringstream ss;
                    ss << "input0, input1, input2, input3, input4, output0, " << input(2)[0] << ", " << y[0] << ", " << y[1] << ", " << 2 * input(0)[1]
                       << ", " << act_enum(gate) << ", nullptr, 0";
                    return call("nnf_mxfp4_grouped_gemm", ss.str());
                }
            };
        } // namespace hip

#define NNF_REGISTER_MX(OPNAME, CLASS)                                                                                            \
    REGISTER_KERNEL_EMITTER(OPNAME, Device(ROCM_GPU).TypeConstraint(element::f32).Tag("nnf_hip_gfx950").Priority(5), CLASS)
        NNF_REGISTER_MX("MxQuantize", hip::MxQuantize)
        NNF_REGISTER_MX("MxDequantize", hip::MxDequantize)
        NNF_REGISTER_MX("MxDot", hip::MxDot)
        NNF_REGISTER_MX("MxGroupedDot", hip::MxGroupedDot)
#undef NNF_REGISTER_MX
    } // namespace kernels
} // namespace nnfusion
