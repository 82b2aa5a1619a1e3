// Kernel emitters of the operators around a mixture's experts and of their products in block-scaled 8-bit floating point
// (fp8_moe_ops.cpp) for ROCM_GPU: each emits a host function around one call into the launcher library, like the emitters on MXFP4
// (mxfp4_emitters.cpp).
#include "../../nnf_fp8_plan.h"
#include "../../nnf_moe_plan.h"
#include "nnf_hip_kernels.h"
#include "nnfusion/core/kernels/hip_gpu/hip_emitter.hpp"
#include "nnfusion/core/kernels/kernel_registration.hpp"
#include "nnfusion/core/operators/generic_op/generic_op.hpp"

#include <climits>
#include <iomanip>

namespace nnfusion
{
    namespace kernels
    {
        namespace hip
        {
            class CallEmitter : public HipLibEmitter
            {
            public:
                using HipLibEmitter::HipLibEmitter;

            protected:
                std::shared_ptr<op::GenericOp> generic() const { return std::dynamic_pointer_cast<op::GenericOp>(m_context->op); }
                op::OpConfig::any& config() const { return generic()->localOpConfig.getRoot(); }
                const Shape& input(size_t i) const { return m_context->inputs[i]->get_shape(); }
                const Shape& output(size_t i) const { return m_context->outputs[i]->get_shape(); }
                // an operator of this kind whose tensors all have elements, and sizes that the calls' ints hold
                bool sized() const
                {
                    if (!generic())
                        return false;
                    for (auto* list : {&m_context->inputs, &m_context->outputs})
                        for (auto& t : *list)
                            for (size_t n : t->get_shape())
                                if (n == 0 || n > (size_t)INT_MAX)
                                    return false;
                    return true;
                }
                bool gate() const { return config()["act"].get<std::string>() == "silu_gate"; }
                static const char* act_enum(bool gate) { return gate ? "NNF_ACT_SILU_GATE" : "NNF_ACT_NONE"; }
                LanguageUnit_p call(const std::string& name, const std::string& arguments, const std::string& ahead = "")
                {
                    LanguageUnit_p lu(new LanguageUnit(get_function_name()));
                    *lu << ahead << "NNF_HIP_CHECK(" << name << "(stream, " << arguments << "));\n";
                    return lu;
                }
            };

            class MoeRoute : public CallEmitter
            {
            public:
                explicit MoeRoute(std::shared_ptr<KernelContext> ctx)
                    : CallEmitter(ctx)
                {
                }
                LanguageUnit_p emit_function_body() override
                {
                    if (!sized())
                        return nullptr;
                    auto& cfg = config();
                    const int tokens = (int)input(0)[0], E = (int)input(0)[1], k = cfg["k"].get<int>(), groups = cfg["groups"].get<int>(),
                              top_groups = cfg["top_groups"].get<int>(), group_top = cfg["group_top"].get<int>();
                    if (!nnf::moe::routable(tokens, E, k, groups, top_groups, group_top))
                        return nullptr;
                    const bool bias = cfg["has_bias"].get<bool>(), live = cfg["has_tokens"].get<bool>();
                    const size_t bytes = nnf::moe::workspace_bytes(tokens, E);
                    std::string ws = "nullptr";
                    if (bytes)
                        ws = allocate_tensor(Shape{bytes}, element::character)->get_name();
                    std::ostringstream routing, ss;
                    routing << "const nnf_moe_routing routing = {" << k << ", "
                            << (cfg["score"].get<std::string>() == "sigmoid" ? "NNF_MOE_SIGMOID" : "NNF_MOE_SOFTMAX") << ", " << groups << ", " << top_groups << ", "
                            << group_top << ", " << (cfg["renormalize"].get<bool>() ? 1 : 0) << ", (float)" << std::setprecision(17) << std::scientific
                            << cfg["scale"].get<double>() << "};\n";
                    ss << "input0, " << (m_context->inputs[0]->get_element_type() == element::f16 ? "NNF_TYPE_F16" : "NNF_TYPE_F32") << ", "
                       << (bias ? "input1" : "nullptr") << ", " << (live ? (bias ? "input2" : "input1") : "nullptr")
                       << ", &routing, output0, output1, output2, output3, output4, " << tokens << ", " << E << ", " << ws << ", " << bytes;
                    return call("nnf_moe_route", ss.str(), routing.str());
                }
            };

            class MoeCombine : public CallEmitter
            {
            public:
                explicit MoeCombine(std::shared_ptr<KernelContext> ctx)
                    : CallEmitter(ctx)
                {
                }
                LanguageUnit_p emit_function_body() override
                {
                    if (!sized() || !nnf::moe::combinable((int)input(1)[0], (int)input(1)[1], (int)input(0)[1]))
                        return nullptr;
                    std::ostringstream ss;
                    ss << "input0, input1, input2, " << (config()["has_residual"].get<bool>() ? "input3" : "nullptr") << ", output0, NNF_TYPE_F16, " << input(1)[0]
                       << ", " << input(0)[0] << ", " << input(1)[1] << ", " << input(0)[1];
                    return call("nnf_moe_combine", ss.str());
                }
            };

            class Fp8Quantize : public CallEmitter
            {
            public:
                explicit Fp8Quantize(std::shared_ptr<KernelContext> ctx)
                    : CallEmitter(ctx)
                {
                }
                LanguageUnit_p emit_function_body() override
                {
                    if (!sized() || !nnf::fp8::convertible((int)output(0)[0], (int)input(0)[1]))
                        return nullptr;
                    std::ostringstream ss;
                    ss << "input0, NNF_TYPE_F16, " << (config()["has_index"].get<bool>() ? "input1" : "nullptr") << ", output0, output1, " << output(0)[0] << ", "
                       << input(0)[0] << ", " << input(0)[1];
                    return call("nnf_fp8_quantize", ss.str());
                }
            };

            class Fp8Dot : public CallEmitter
            {
            public:
                explicit Fp8Dot(std::shared_ptr<KernelContext> ctx)
                    : CallEmitter(ctx)
                {
                }
                LanguageUnit_p emit_function_body() override
                {
                    if (!sized())
                        return nullptr;
                    const bool bias = config()["has_bias"].get<bool>(), residual = config()["has_residual"].get<bool>();
                    const Shape& y = output(0);
                    // what the launcher declines
                    if ((gate() && (bias || residual)) || !nnf::fp8::servable((int)y[0], (int)y[1], (int)input(0)[1], gate(), 0))
                        return nullptr;
                    std::ostringstream ss;
                    ss << "input0, input1, input2, input3, output0, NNF_TYPE_F16, " << y[0] << ", " << y[1] << ", " << input(0)[1] << ", "
                       << (bias ? "input4" : "nullptr") << ", " << (residual ? (bias ? "input5" : "input4") : "nullptr") << ", " << act_enum(gate());
                    return call("nnf_fp8_gemm", ss.str());
                }
            };

            class Fp8GroupedDot : public CallEmitter
            {
            public:
                explicit Fp8GroupedDot(std::shared_ptr<KernelContext> ctx)
                    : CallEmitter(ctx)
                {
                }
                LanguageUnit_p emit_function_body() override
                {
                    if (!sized())
                        return nullptr;
                    const Shape& y = output(0);
                    if (!nnf::fp8::servable((int)y[0], (int)y[1], (int)input(0)[1], gate(), (int)input(2)[0]))
                        return nullptr;
                    std::ostringstream ss;
                    ss << "input0, input1, input2, input3, input4, output0, NNF_TYPE_F16, " << input(2)[0] << ", " << y[0] << ", " << y[1] << ", " << input(0)[1]
                       << ", " << act_enum(gate());
                    return call("nnf_fp8_grouped_gemm", ss.str());
                }
            };
        } // namespace hip

#define NNF_REGISTER_CALL(OPNAME, CLASS)                                                                                          \
    REGISTER_KERNEL_EMITTER(OPNAME, Device(ROCM_GPU).TypeConstraint(element::f32).Tag("nnf_hip_gfx950").Priority(5), CLASS)
        NNF_REGISTER_CALL("MoeRoute", hip::MoeRoute)
        NNF_REGISTER_CALL("MoeCombine", hip::MoeCombine)
        NNF_REGISTER_CALL("Fp8Quantize", hip::Fp8Quantize)
        NNF_REGISTER_CALL("Fp8Dot", hip::Fp8Dot)
        NNF_REGISTER_CALL("Fp8GroupedDot", hip::Fp8GroupedDot)
#undef NNF_REGISTER_CALL
    } // namespace kernels
} // namespace nnfusion
