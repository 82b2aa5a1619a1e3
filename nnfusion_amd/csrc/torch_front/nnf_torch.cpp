// The per-call path of nnfusion_amd/ops.py: torch tensors in, one call of the C ABI (include/nnf_hip_kernels.h) out.
//
// A decode step is a run of kernels of 4 - 11 us each; the same calls through ctypes (argument checks, sizes and pointers
// taken from the tensors one Python attribute at a time, a foreign call of up to twenty converted arguments) took the host
// 10 - 13 us apiece, so that a step of twelve calls was bound by the interpreter.  Here a call checks its tensors, allocates
// what the caller did not bring and enters the library in about a microsecond.  No state is kept between calls.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <c10/hip/HIPStream.h>

#include "../nnf_moe_plan.h"
#include "nnf_hip_kernels.h"

namespace
{
    using at::Tensor;

    PyObject* g_error = nullptr; // nnfusion_amd.ops.NnfError(status, where)

    // thrown with the Python error set
    struct Raised
    {
    };
    [[noreturn]] void raise(PyObject* type, const char* text)
    {
        PyErr_SetString(type, text);
        throw Raised();
    }
    void require(bool ok, const char* text)
    {
        if (!ok)
            raise(PyExc_AssertionError, text);
    }
    // the library's error
    [[noreturn]] void fail(const char* where, int status)
    {
        PyObject* const e = g_error ? PyObject_CallFunction(g_error, "is", status, where) : nullptr;
        if (e)
            PyErr_SetObject(g_error, e);
        Py_XDECREF(e);
        throw Raised();
    }
    // one call of the library, the interpreter released meanwhile (a launch into a full queue waits)
    template <typename F, typename... Args>
    void call(const char* where, F* function, Args... args)
    {
        PyThreadState* const thread = PyEval_SaveThread();
        const int status = function(args...);
        PyEval_RestoreThread(thread);
        if (status != NNF_OK)
            fail(where, status);
    }

    const Tensor& tensor(PyObject* o)
    {
        if (!THPVariable_Check(o))
            raise(PyExc_TypeError, "a torch.Tensor is expected");
        return THPVariable_Unpack(o);
    }
    // the address of a tensor, or null for None
    void* address(PyObject* o) { return o == Py_None ? nullptr : tensor(o).data_ptr(); }
    int integer(PyObject* o)
    {
        const long v = PyLong_AsLong(o);
        if (v == -1 && PyErr_Occurred())
            throw Raised();
        if (v != (int)v)
            raise(PyExc_OverflowError, "integer argument out of range");
        return (int)v;
    }
    float real(PyObject* o)
    {
        const double v = PyFloat_AsDouble(o);
        if (v == -1.0 && PyErr_Occurred())
            throw Raised();
        return (float)v;
    }
    void matrix(const Tensor& t)
    {
        if (t.dim() != 2)
            raise(PyExc_ValueError, "a matrix is expected");
    }
    nnf_stream_t stream() { return (nnf_stream_t)c10::hip::getCurrentHIPStream().stream(); }

    // The caller's output buffer, or a new one.  `object`: what the Python caller gets back
    struct Output
    {
        PyObject* object = nullptr;
        void* data = nullptr;
        Output(PyObject* given, int m, int n, at::ScalarType type, const Tensor& like)
        {
            if (given != Py_None)
            {
                data = tensor(given).data_ptr();
                Py_INCREF(given);
                object = given;
                return;
            }
            Tensor t = at::empty({m, n}, like.options().dtype(type));
            data = t.data_ptr();
            object = THPVariable_Wrap(std::move(t));
            if (!object)
                throw Raised();
        }
        ~Output() { Py_XDECREF(object); }
        PyObject* release()
        {
            PyObject* o = object;
            object = nullptr;
            return o;
        }
    };
    // The caller's workspace, or one of `need()` bytes for this call (torch's allocator keeps the block for the next)
    struct Workspace
    {
        Tensor own;
        void* data = nullptr;
        size_t bytes = 0;
        template <typename F>
        Workspace(PyObject* given, const Tensor& like, F need, size_t least = 16)
        {
            if (given != Py_None)
            {
                const Tensor& t = tensor(given);
                data = t.data_ptr();
                bytes = (size_t)t.numel();
                return;
            }
            const size_t n = need();
            bytes = n > least ? n : least;
            if (!bytes)
                return;
            own = at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
            data = own.data_ptr();
        }
    };
    // nnf_plan with nothing but the synchronisation words, or a null pointer where the caller passed none
    struct SyncPlan
    {
        nnf_plan plan = {};
        const nnf_plan* ptr = nullptr;
        SyncPlan(PyObject* sync, int spin_limit = 0)
        {
            if (sync == Py_None)
                return;
            const Tensor& t = tensor(sync);
            plan.sync_flags = t.data_ptr();
            plan.sync_flags_bytes = (size_t)t.nbytes();
            plan.spin_limit = spin_limit;
            ptr = &plan;
        }
    };
    nnf_quant quant(PyObject* bits, PyObject* group, PyObject* zp, PyObject* zero_points)
    {
        return nnf_quant{integer(bits), integer(group), integer(zp), address(zero_points)};
    }

    using Args = PyObject* const*;

    // (a, wq, scales, group, zp, out, workspace)
    PyObject* w4a16_gemm(Args v)
    {
        const Tensor &a = tensor(v[0]), &wq = tensor(v[1]), &s = tensor(v[2]);
        matrix(a), matrix(wq), matrix(s);
        const int m = (int)a.size(0), k = (int)a.size(1), n = (int)wq.size(0), group = integer(v[3]);
        require(a.scalar_type() == at::kHalf && wq.scalar_type() == at::kByte && s.scalar_type() == at::kHalf, "fp16 activations, uint8 weights, fp16 scales");
        require(a.is_contiguous() && wq.is_contiguous() && s.is_contiguous(), "contiguous operands");
        require(group > 0 && wq.size(1) * 2 == k && s.size(0) == n && s.size(1) == k / group, "shapes of weights and scales");
        Output y(v[5], m, n, at::kHalf, a);
        Workspace w(v[6], a, [&] { return nnf_w4a16_gemm_workspace_bytes(m, n, k, group); });
        call("nnf_w4a16_gemm", nnf_w4a16_gemm, stream(), a.data_ptr(), wq.data_ptr(), s.data_ptr(), y.data, m, n, k, group, integer(v[4]),
             w.data, w.bytes);
        return y.release();
    }

    // (a, wq, scales, bits, group, zp, zero_points, out, workspace, sync, spin_limit)
    PyObject* wna16_gemm(Args v)
    {
        const Tensor &a = tensor(v[0]), &wq = tensor(v[1]), &s = tensor(v[2]);
        matrix(a), matrix(wq), matrix(s);
        const int m = (int)a.size(0), k = (int)a.size(1), n = (int)wq.size(0);
        const nnf_quant q = quant(v[3], v[4], v[5], v[6]);
        require(a.scalar_type() == at::kHalf && wq.scalar_type() == at::kByte && s.scalar_type() == at::kHalf, "fp16 activations, uint8 weights, fp16 scales");
        require(a.is_contiguous() && wq.is_contiguous() && s.is_contiguous(), "contiguous operands");
        require(q.group > 0 && wq.size(1) * 8 == (int64_t)k * q.bits && s.size(0) == n && s.size(1) == k / q.group, "shapes of weights and scales");
        if (q.zero_points)
        {
            const Tensor& z = tensor(v[6]);
            require(z.scalar_type() == at::kByte && z.is_contiguous(), "zero points: contiguous uint8");
            require(z.dim() == 2 && z.size(0) == n && z.size(1) == (k / q.group * q.bits + 7) / 8, "shape of the zero points");
        }
        Output y(v[7], m, n, at::kHalf, a);
        Workspace w(v[8], a, [&] { return nnf_wna16_gemm_preferred_workspace_bytes(m, n, k, &q); });
        const SyncPlan plan(v[9], integer(v[10]));
        call(plan.ptr ? "nnf_wna16_gemm_planned" : "nnf_wna16_gemm", nnf_wna16_gemm_planned, stream(), a.data_ptr(), wq.data_ptr(),
             s.data_ptr(), y.data, m, n, k, &q, plan.ptr, w.data, w.bytes);
        return y.release();
    }

    // (a, wq, scales, group, zp, rms_gamma, rms_eps, bias, residual, act, out, workspace, sync, spin_limit)
    PyObject* w4a16_gemm_fused(Args v)
    {
        const Tensor &a = tensor(v[0]), &wq = tensor(v[1]), &s = tensor(v[2]);
        matrix(a);
        const int m = (int)a.size(0), k = (int)a.size(1), group = integer(v[3]), zp = integer(v[4]), act = integer(v[9]);
        const int rows = (int)wq.size(0), n = rows / (act == NNF_ACT_SILU_GATE ? 2 : 1);
        Output y(v[10], m, n, at::kHalf, a);
        const SyncPlan plan(v[12], integer(v[13]));
        Workspace w(v[11], a, [&] {
            const size_t need = nnf_w4a16_gemm_fused_workspace_bytes(m, n, k, group, act);
            return plan.ptr ? need + nnf_w4a16_gemm_variant_workspace_bytes(m, rows, k, group, NNF_W4A16_AUTO, plan.ptr) : need;
        });
        call(plan.ptr ? "nnf_w4a16_gemm_fused_variant" : "nnf_w4a16_gemm_fused", nnf_w4a16_gemm_fused_variant, stream(), a.data_ptr(),
             wq.data_ptr(), s.data_ptr(), y.data, m, n, k, group, zp, address(v[5]), real(v[6]), address(v[7]), address(v[8]), act,
             NNF_W4A16_AUTO, plan.ptr, w.data, w.bytes);
        return y.release();
    }

    // (x, gamma, wgu, sgu, wd, sd, eps, group, zp, out, workspace, sync, spin_limit)
    PyObject* fused_mlp_w4a16(Args v)
    {
        const Tensor& x = tensor(v[0]);
        matrix(x);
        const int m = (int)x.size(0), h = (int)x.size(1), i = (int)(tensor(v[2]).size(0) / 2), group = integer(v[7]);
        Output y(v[9], m, h, at::kHalf, x);
        Workspace w(v[10], x, [&] { return nnf_fused_mlp_w4a16_workspace_bytes(m, h, i, group); });
        const SyncPlan plan(v[11], integer(v[12]));
        call(plan.ptr ? "nnf_fused_mlp_w4a16_planned" : "nnf_fused_mlp_w4a16", nnf_fused_mlp_w4a16_planned, stream(), x.data_ptr(),
             address(v[1]), real(v[6]), address(v[2]), address(v[3]), address(v[4]), address(v[5]), y.data, m, h, i, group, integer(v[8]),
             plan.ptr, plan.ptr, w.data, w.bytes);
        return y.release();
    }

    // (a, wq, scales, bits, group, zp, zero_points, rms_gamma, rms_eps, bias, residual, act, out, workspace)
    PyObject* wna16_gemm_fused(Args v)
    {
        const Tensor &a = tensor(v[0]), &wq = tensor(v[1]), &s = tensor(v[2]);
        matrix(a);
        const int m = (int)a.size(0), k = (int)a.size(1), act = integer(v[11]), n = (int)(wq.size(0) / (act == NNF_ACT_SILU_GATE ? 2 : 1));
        const nnf_quant q = quant(v[3], v[4], v[5], v[6]);
        Output y(v[12], m, n, at::kHalf, a);
        Workspace w(v[13], a, [&] { return nnf_wna16_gemm_fused_workspace_bytes(m, n, k, &q, act); });
        call("nnf_wna16_gemm_fused", nnf_wna16_gemm_fused, stream(), a.data_ptr(), wq.data_ptr(), s.data_ptr(), y.data, m, n, k, &q,
             address(v[7]), real(v[8]), address(v[9]), address(v[10]), act, w.data, w.bytes);
        return y.release();
    }

    // (x, gamma, wgu, sgu, wd, sd, bits, group, zp, zgu, zd, eps, out, workspace)
    PyObject* fused_mlp_wna16(Args v)
    {
        const Tensor& x = tensor(v[0]);
        matrix(x);
        const int m = (int)x.size(0), h = (int)x.size(1), i = (int)(tensor(v[2]).size(0) / 2);
        const nnf_quant qa = quant(v[6], v[7], v[8], v[9]), qb = quant(v[6], v[7], v[8], v[10]);
        Output y(v[12], m, h, at::kHalf, x);
        Workspace w(v[13], x, [&] { return nnf_fused_mlp_wna16_workspace_bytes(m, h, i, &qa, &qb); });
        call("nnf_fused_mlp_wna16", nnf_fused_mlp_wna16, stream(), x.data_ptr(), address(v[1]), real(v[11]), address(v[2]), address(v[3]),
             address(v[4]), address(v[5]), y.data, m, h, i, &qa, &qb, w.data, w.bytes);
        return y.release();
    }

    // the raw int32 accumulators (no scales) or the fp16 product
    PyObject* w8a8(const Tensor& a, const Tensor& b, const Tensor* s_tok, const Tensor* s_ch, PyObject* out, PyObject* workspace, PyObject* sync)
    {
        matrix(a), matrix(b);
        const int m = (int)a.size(0), k = (int)a.size(1), n = (int)b.size(0);
        const bool raw = !s_tok;
        require(a.scalar_type() == at::kChar && b.scalar_type() == at::kChar, "int8 operands");
        if (!raw)
            require(s_tok->scalar_type() == at::kFloat && s_ch->scalar_type() == at::kFloat, "fp32 scales");
        Output y(out, m, n, raw ? at::kInt : at::kHalf, a);
        const SyncPlan plan(sync);
        Workspace w(workspace, a, [&] {
            return plan.ptr ? nnf_w8a8_gemm_variant_workspace_bytes(m, n, k, NNF_W8A8_AUTO, plan.ptr) : nnf_w8a8_gemm_workspace_bytes(m, n, k);
        });
        call(plan.ptr ? "nnf_w8a8_gemm_variant" : raw ? "nnf_w8a8_gemm_acc" : "nnf_w8a8_gemm", nnf_w8a8_gemm_variant, stream(),
             a.data_ptr(), raw ? nullptr : s_tok->data_ptr(), b.data_ptr(), raw ? nullptr : s_ch->data_ptr(), raw ? nullptr : y.data,
             raw ? y.data : nullptr, m, n, k, NNF_W8A8_AUTO, plan.ptr, w.data, w.bytes);
        return y.release();
    }
    // (a, s_tok, w, s_ch, out, workspace, sync)
    PyObject* w8a8_gemm(Args v) { return w8a8(tensor(v[0]), tensor(v[2]), &tensor(v[1]), &tensor(v[3]), v[4], v[5], v[6]); }
    // (a, w, out, workspace, sync)
    PyObject* w8a8_gemm_acc(Args v) { return w8a8(tensor(v[0]), tensor(v[1]), nullptr, nullptr, v[2], v[3], v[4]); }

    // (op, a, b, out)
    PyObject* elementwise(Args v)
    {
        const Tensor& a = tensor(v[1]);
        require(a.scalar_type() == at::kHalf && a.is_contiguous(), "a contiguous fp16 tensor");
        const int64_t cols = a.size(-1);
        const size_t rows = cols ? (size_t)(a.numel() / cols) : 0;
        int b_is_row = 0;
        if (v[2] != Py_None)
        {
            const Tensor& b = tensor(v[2]);
            require(b.scalar_type() == at::kHalf && b.is_contiguous(), "a contiguous fp16 second operand");
            b_is_row = b.dim() == 1 && a.dim() > 1;
            require(b_is_row || b.sizes() == a.sizes(), "operands of one shape");
        }
        PyObject* out = v[3];
        if (out == Py_None)
        {
            out = THPVariable_Wrap(at::empty_like(a));
            if (!out)
                throw Raised();
        }
        else
            Py_INCREF(out);
        try
        {
            call("nnf_elementwise_f16", nnf_elementwise_f16, stream(), integer(v[0]), a.data_ptr(), address(v[2]), tensor(out).data_ptr(),
                 rows, (int)cols, b_is_row);
        }
        catch (...)
        {
            Py_DECREF(out);
            throw;
        }
        return out;
    }

    // (x, gamma, eps, out)
    PyObject* rms_norm(Args v)
    {
        const Tensor& x = tensor(v[0]);
        matrix(x);
        const int m = (int)x.size(0), k = (int)x.size(1);
        Output y(v[3], m, k, x.scalar_type(), x);
        call("nnf_rms_norm_f16", nnf_rms_norm_f16, stream(), x.data_ptr(), address(v[1]), y.data, m, k, real(v[2]));
        return y.release();
    }

    // (wq, scales, bits, group, zp, zero_points, out)
    PyObject* dequantize(Args v)
    {
        const Tensor& wq = tensor(v[0]);
        matrix(wq);
        const nnf_quant q = quant(v[2], v[3], v[4], v[5]);
        require(q.bits > 0, "bits of the weights");
        const int n = (int)wq.size(0), k = (int)(wq.size(1) * 8 / q.bits);
        Output y(v[6], n, k, at::kHalf, wq);
        call("nnf_dequantize_f16", nnf_dequantize_f16, stream(), wq.data_ptr(), address(v[1]), y.data, n, k, &q);
        return y.release();
    }

    // ---- MXFP4.  These calls run on the device that holds their first tensor, whichever is current, on its current stream
    bool is(const Tensor& t, at::ScalarType type, std::initializer_list<int64_t> sizes)
    {
        return t.scalar_type() == type && t.is_contiguous() && t.sizes() == at::IntArrayRef(sizes.begin(), sizes.size());
    }
    void on_device(const Tensor& first, std::initializer_list<PyObject*> others)
    {
        require(first.is_cuda(), "tensors on a GPU");
        for (PyObject* o : others)
            require(o == Py_None || tensor(o).device() == first.device(), "all tensors on one device");
    }
    int size32(int64_t v)
    {
        if (v != (int)v)
            raise(PyExc_OverflowError, "size out of range");
        return (int)v;
    }
    // a new tensor of these sizes where the caller brought none; either way a reference of its own
    PyObject* output(PyObject* given, std::initializer_list<int64_t> sizes, at::ScalarType type, const Tensor& like, const char* text)
    {
        if (given == Py_None)
        {
            // (through the dispatcher, 0.25 us: modes see it, and deterministic ones fill it)
            PyObject* const o = THPVariable_Wrap(at::empty(at::IntArrayRef(sizes.begin(), sizes.size()), like.options().dtype(type)));
            if (!o)
                throw Raised();
            return o;
        }
        require(is(tensor(given), type, sizes), text);
        Py_INCREF(given);
        return given;
    }
    struct Owned
    {
        PyObject* object;
        explicit Owned(PyObject* o)
            : object(o)
        {
        }
        Owned(const Owned&) = delete;
        ~Owned() { Py_XDECREF(object); }
        void* data() const { return THPVariable_Unpack(object).data_ptr(); }
        PyObject* release()
        {
            PyObject* o = object;
            object = nullptr;
            return o;
        }
    };
    // (no MXFP4 kernel needs a workspace: none is allocated for a caller that brings none)
    size_t bytes_of(PyObject* o) { return o == Py_None ? 0 : (size_t)tensor(o).nbytes(); }
    void workspace_checked(PyObject* o) { require(o == Py_None || (tensor(o).scalar_type() == at::kByte && tensor(o).is_contiguous()), "workspace: contiguous uint8"); }

    // (x, rows, codes, scales) -> (codes, scales)
    PyObject* mxfp4_quantize(Args v)
    {
        const Tensor& x = tensor(v[0]);
        matrix(x);
        require(x.scalar_type() == at::kHalf && x.is_contiguous(), "a contiguous fp16 matrix");
        const int source = size32(x.size(0)), k = size32(x.size(1));
        int rows = source;
        if (v[1] != Py_None)
        {
            const Tensor& index = tensor(v[1]);
            require(index.scalar_type() == at::kInt && index.dim() == 1 && index.is_contiguous(), "rows: a contiguous int32 vector");
            rows = size32(index.size(0));
        }
        for (int i = 2; i < 4; ++i)
            if (v[i] != Py_None)
                require(is(tensor(v[i]), at::kByte, {rows, i == 2 ? k / 2 : nnf_mxfp4_scale_bytes(k)}), i == 2 ? "codes: contiguous uint8 [rows, K/2]" : "scales: contiguous uint8 [rows, mxfp4_scale_bytes(K)]");
        on_device(x, {v[1], v[2], v[3]});
        const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
        Owned codes(output(v[2], {rows, k / 2}, at::kByte, x, "codes")), scales(output(v[3], {rows, nnf_mxfp4_scale_bytes(k)}, at::kByte, x, "scales"));
        call("nnf_mxfp4_quantize_f16", nnf_mxfp4_quantize_f16, stream(), x.data_ptr(), address(v[1]), codes.data(), scales.data(), rows, source, k);
        PyObject* const both = PyTuple_Pack(2, codes.object, scales.object);
        if (!both)
            throw Raised();
        return both;
    }

    // (codes, scales, out)
    PyObject* mxfp4_dequantize(Args v)
    {
        const Tensor &codes = tensor(v[0]), &scales = tensor(v[1]);
        matrix(codes);
        const int rows = size32(codes.size(0)), k = size32(codes.size(1) * 2);
        require(is(codes, at::kByte, {rows, k / 2}), "codes: contiguous uint8 [rows, K/2]");
        require(is(scales, at::kByte, {rows, nnf_mxfp4_scale_bytes(k)}), "scales: contiguous uint8 [rows, mxfp4_scale_bytes(K)]");
        if (v[2] != Py_None)
            require(is(tensor(v[2]), at::kHalf, {rows, k}), "out: contiguous fp16 [rows, K]");
        on_device(codes, {v[1], v[2]});
        const c10::hip::HIPGuardMasqueradingAsCUDA guard(codes.device());
        Owned y(output(v[2], {rows, k}, at::kHalf, codes, "out"));
        call("nnf_mxfp4_dequantize_f16", nnf_mxfp4_dequantize_f16, stream(), codes.data_ptr(), scales.data_ptr(), y.data(), rows, k);
        return y.release();
    }

    // the activations of either product: codes [M, K/2] and their scale bytes
    void mxfp4_activations(const Tensor& a, const Tensor& as, int& m, int& k)
    {
        matrix(a);
        m = size32(a.size(0)), k = size32(a.size(1) * 2);
        require(is(a, at::kByte, {m, k / 2}), "activations: contiguous uint8 [M, K/2]");
        require(is(as, at::kByte, {m, nnf_mxfp4_scale_bytes(k)}), "scales of the activations: contiguous uint8 [M, mxfp4_scale_bytes(K)]");
    }
    // columns of Y from the rows of a weight matrix
    int mxfp4_columns(int64_t rows, int act)
    {
        require(act == NNF_ACT_NONE || act == NNF_ACT_SILU_GATE, "act: 0, or 1 for SiLU-gate");
        require(act == NNF_ACT_NONE || rows % 2 == 0, "gate rows and as many up rows");
        return size32(act == NNF_ACT_SILU_GATE ? rows / 2 : rows);
    }

    // (a, a_scales, w, w_scales, bias, residual, act, out, workspace, variant)
    PyObject* mxfp4_gemm(Args v)
    {
        const Tensor &a = tensor(v[0]), &as = tensor(v[1]), &w = tensor(v[2]), &ws = tensor(v[3]);
        int m, k;
        mxfp4_activations(a, as, m, k);
        matrix(w);
        const int act = integer(v[6]), n = mxfp4_columns(w.size(0), act);
        require(is(w, at::kByte, {w.size(0), k / 2}) && is(ws, at::kByte, {w.size(0), nnf_mxfp4_scale_bytes(k)}), "weights: contiguous uint8 [N, K/2], scales [N, mxfp4_scale_bytes(K)]");
        if (v[4] != Py_None)
            require(is(tensor(v[4]), at::kHalf, {n}), "bias: contiguous fp16 [N]");
        if (v[5] != Py_None)
            require(is(tensor(v[5]), at::kHalf, {m, n}), "residual: contiguous fp16 [M, N]");
        if (v[7] != Py_None)
            require(is(tensor(v[7]), at::kHalf, {m, n}), "out: contiguous fp16 [M, N]");
        workspace_checked(v[8]);
        on_device(a, {v[1], v[2], v[3], v[4], v[5], v[7], v[8]});
        const c10::hip::HIPGuardMasqueradingAsCUDA guard(a.device());
        Owned y(output(v[7], {m, n}, at::kHalf, a, "out"));
        call("nnf_mxfp4_gemm", nnf_mxfp4_gemm_variant, stream(), a.data_ptr(), as.data_ptr(), w.data_ptr(), ws.data_ptr(), y.data(), m, n, k, address(v[4]),
             address(v[5]), act, integer(v[9]), address(v[8]), bytes_of(v[8]));
        return y.release();
    }

    // (a, a_scales, w, w_scales, offsets, act, out, workspace, variant)
    PyObject* mxfp4_grouped_gemm(Args v)
    {
        const Tensor &a = tensor(v[0]), &as = tensor(v[1]), &w = tensor(v[2]), &ws = tensor(v[3]), &offsets = tensor(v[4]);
        int m, k;
        mxfp4_activations(a, as, m, k);
        if (w.dim() != 3)
            raise(PyExc_ValueError, "weights [experts, N, K/2] are expected");
        const int experts = size32(w.size(0)), act = integer(v[5]), n = mxfp4_columns(w.size(1), act);
        require(is(w, at::kByte, {experts, w.size(1), k / 2}) && is(ws, at::kByte, {experts, w.size(1), nnf_mxfp4_scale_bytes(k)}),
                "weights: contiguous uint8 [experts, N, K/2], scales [experts, N, mxfp4_scale_bytes(K)]");
        require(is(offsets, at::kInt, {(int64_t)experts + 1}), "offsets: contiguous int32 [experts + 1]");
        if (v[6] != Py_None)
            require(is(tensor(v[6]), at::kHalf, {m, n}), "out: contiguous fp16 [M, N]");
        workspace_checked(v[7]);
        on_device(a, {v[1], v[2], v[3], v[4], v[6], v[7]});
        const c10::hip::HIPGuardMasqueradingAsCUDA guard(a.device());
        Owned y(output(v[6], {m, n}, at::kHalf, a, "out"));
        call("nnf_mxfp4_grouped_gemm", nnf_mxfp4_grouped_gemm_variant, stream(), a.data_ptr(), as.data_ptr(), w.data_ptr(), ws.data_ptr(), offsets.data_ptr(),
             y.data(), experts, m, n, k, act, integer(v[8]), address(v[7]), bytes_of(v[7]));
        return y.release();
    }

    // ---- routing and combining, on the device that holds their first tensor too
    bool truth(PyObject* o)
    {
        const int v = PyObject_IsTrue(o);
        if (v < 0)
            throw Raised();
        return v != 0;
    }
    int type_of(const Tensor& t, bool wide, const char* text)
    {
        if (t.scalar_type() == at::kHalf)
            return NNF_TYPE_F16;
        if (t.scalar_type() == at::kBFloat16)
            return NNF_TYPE_BF16;
        require(wide && t.scalar_type() == at::kFloat, text);
        return NNF_TYPE_F32;
    }

    // (logits, k, score, bias, groups, top_groups, group_top, renormalize, scale, tokens, out, workspace) -> (weights, experts, rows, offsets, positions)
    PyObject* moe_route(Args v)
    {
        const Tensor& logits = tensor(v[0]);
        matrix(logits);
        require(logits.is_contiguous(), "contiguous logits [tokens, experts]");
        const int type = type_of(logits, true, "logits: fp16, bf16 or fp32"), tokens = size32(logits.size(0)), E = size32(logits.size(1));
        const nnf_moe_routing routing = {integer(v[1]), integer(v[2]), integer(v[4]), integer(v[5]), integer(v[6]), truth(v[7]), real(v[8])};
        require(routing.k > 0 && routing.k <= E, "k: at least 1, at most the experts there are"); // (ahead of results of that size)
        const int64_t k = routing.k, pairs = tokens * k;
        if (pairs > nnf::moe::MAX_PAIRS) // (likewise)
            fail("nnf_moe_route", NNF_ERR_UNSUPPORTED_SHAPE);
        if (v[3] != Py_None)
            require(is(tensor(v[3]), at::kFloat, {E}), "bias: contiguous fp32 [experts]");
        if (v[9] != Py_None)
            require(tensor(v[9]).scalar_type() == at::kInt && tensor(v[9]).numel() == 1, "tokens: one int32");
        PyObject* given[5] = {Py_None, Py_None, Py_None, Py_None, Py_None};
        if (v[10] != Py_None)
        {
            require(PyTuple_Check(v[10]) && PyTuple_GET_SIZE(v[10]) == 5, "out: (weights, experts, rows, offsets, positions)");
            for (int i = 0; i < 5; ++i)
                given[i] = PyTuple_GET_ITEM(v[10], i);
        }
        if (given[0] != Py_None)
            require(is(tensor(given[0]), at::kFloat, {tokens, k}), "weights: contiguous fp32 [tokens, k]");
        if (given[1] != Py_None)
            require(is(tensor(given[1]), at::kInt, {tokens, k}), "experts: contiguous int32 [tokens, k]");
        if (given[2] != Py_None)
            require(is(tensor(given[2]), at::kInt, {pairs}), "rows: contiguous int32 [tokens * k]");
        if (given[3] != Py_None)
            require(is(tensor(given[3]), at::kInt, {(int64_t)E + 1}), "offsets: contiguous int32 [experts + 1]");
        if (given[4] != Py_None)
            require(is(tensor(given[4]), at::kInt, {tokens, k}), "positions: contiguous int32 [tokens, k]");
        workspace_checked(v[11]);
        on_device(logits, {v[3], v[9], given[0], given[1], given[2], given[3], given[4], v[11]});
        const c10::hip::HIPGuardMasqueradingAsCUDA guard(logits.device());
        const Owned weights(output(given[0], {tokens, k}, at::kFloat, logits, "weights")), experts(output(given[1], {tokens, k}, at::kInt, logits, "experts")),
            rows(output(given[2], {pairs}, at::kInt, logits, "rows")), offsets(output(given[3], {(int64_t)E + 1}, at::kInt, logits, "offsets")),
            positions(output(given[4], {tokens, k}, at::kInt, logits, "positions"));
        const Workspace w(v[11], logits, [&] { return nnf_moe_route_workspace_bytes(tokens, E, routing.k); }, 0);
        call("nnf_moe_route", nnf_moe_route, stream(), logits.data_ptr(), type, address(v[3]), address(v[9]), &routing, weights.data(), experts.data(), rows.data(),
             offsets.data(), positions.data(), tokens, E, w.data, w.bytes);
        PyObject* const all = PyTuple_Pack(5, weights.object, experts.object, rows.object, offsets.object, positions.object);
        if (!all)
            throw Raised();
        return all;
    }

    // (x, weights, positions, residual, out)
    PyObject* moe_combine(Args v)
    {
        const Tensor &x = tensor(v[0]), &weights = tensor(v[1]), &positions = tensor(v[2]);
        matrix(x), matrix(weights);
        const int type = type_of(x, false, "x: fp16 or bf16"), rows = size32(x.size(0)), n = size32(x.size(1)), tokens = size32(weights.size(0)), k = size32(weights.size(1));
        require(x.is_contiguous(), "contiguous x [rows, N]");
        require(is(weights, at::kFloat, {tokens, k}), "weights: contiguous fp32 [tokens, k]");
        require(is(positions, at::kInt, {tokens, k}), "positions: contiguous int32 [tokens, k]");
        if (v[3] != Py_None)
            require(is(tensor(v[3]), x.scalar_type(), {tokens, n}), "residual: contiguous [tokens, N] of x's type");
        if (v[4] != Py_None)
            require(is(tensor(v[4]), x.scalar_type(), {tokens, n}), "out: contiguous [tokens, N] of x's type");
        on_device(x, {v[1], v[2], v[3], v[4]});
        const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
        Owned y(output(v[4], {tokens, n}, x.scalar_type(), x, "out"));
        call("nnf_moe_combine", nnf_moe_combine, stream(), x.data_ptr(), weights.data_ptr(), positions.data_ptr(), address(v[3]), y.data(), type, tokens, rows, k, n);
        return y.release();
    }

    // ---- block-scaled 8-bit floating point, likewise
    constexpr auto E4M3 = at::kFloat8_e4m3fn;
    int64_t blocks128(int64_t size) { return (size + 127) / 128; }
    PyObject* pair(const Owned& a, const Owned& b)
    {
        PyObject* const both = PyTuple_Pack(2, a.object, b.object);
        if (!both)
            throw Raised();
        return both;
    }

    // (x, rows, codes, scales) -> (codes, scales)
    PyObject* fp8_quantize(Args v)
    {
        const Tensor& x = tensor(v[0]);
        matrix(x);
        const int type = type_of(x, false, "x: fp16 or bf16");
        require(x.is_contiguous(), "a contiguous matrix");
        const int source = size32(x.size(0)), k = size32(x.size(1));
        int rows = source;
        if (v[1] != Py_None)
        {
            const Tensor& index = tensor(v[1]);
            require(index.scalar_type() == at::kInt && index.dim() == 1 && index.is_contiguous(), "rows: a contiguous int32 vector");
            rows = size32(index.size(0));
        }
        if (v[2] != Py_None)
            require(is(tensor(v[2]), E4M3, {rows, k}), "codes: contiguous float8_e4m3fn [rows, K]");
        if (v[3] != Py_None)
            require(is(tensor(v[3]), at::kFloat, {blocks128(k), rows}), "scales: contiguous fp32 [ceil(K/128), rows]");
        on_device(x, {v[1], v[2], v[3]});
        const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
        const Owned codes(output(v[2], {rows, k}, E4M3, x, "codes")), scales(output(v[3], {blocks128(k), rows}, at::kFloat, x, "scales"));
        call("nnf_fp8_quantize", nnf_fp8_quantize, stream(), x.data_ptr(), type, address(v[1]), codes.data(), scales.data(), rows, source, k);
        return pair(codes, scales);
    }

    // (w, codes, scales) -> (codes, scales)
    PyObject* fp8_quantize_weights(Args v)
    {
        const Tensor& w = tensor(v[0]);
        if (w.dim() != 2 && w.dim() != 3)
            raise(PyExc_ValueError, "weights [N, K] or [matrices, N, K] are expected");
        const int type = type_of(w, false, "w: fp16 or bf16");
        require(w.is_contiguous(), "contiguous weights");
        const bool many = w.dim() == 3;
        const int matrices = many ? size32(w.size(0)) : 1, n = size32(w.size(-2)), k = size32(w.size(-1));
        const int64_t nb = blocks128(n), kb = blocks128(k);
        if (v[1] != Py_None)
            require(tensor(v[1]).scalar_type() == E4M3 && tensor(v[1]).is_contiguous() && tensor(v[1]).sizes() == w.sizes(), "codes: contiguous float8_e4m3fn of w's shape");
        if (v[2] != Py_None)
            require(many ? is(tensor(v[2]), at::kFloat, {matrices, nb, kb}) : is(tensor(v[2]), at::kFloat, {nb, kb}), "scales: contiguous fp32 [.., ceil(N/128), ceil(K/128)]");
        on_device(w, {v[1], v[2]});
        const c10::hip::HIPGuardMasqueradingAsCUDA guard(w.device());
        const Owned codes(many ? output(v[1], {matrices, n, k}, E4M3, w, "codes") : output(v[1], {n, k}, E4M3, w, "codes"));
        const Owned scales(many ? output(v[2], {matrices, nb, kb}, at::kFloat, w, "scales") : output(v[2], {nb, kb}, at::kFloat, w, "scales"));
        call("nnf_fp8_quantize_weights", nnf_fp8_quantize_weights, stream(), w.data_ptr(), type, codes.data(), scales.data(), matrices, n, k);
        return pair(codes, scales);
    }

    // the type of a product's result: that of the first tensor given, or the one named, or fp16
    at::ScalarType fp8_result(std::initializer_list<PyObject*> tensors, PyObject* dtype)
    {
        at::ScalarType type = at::kHalf;
        bool known = dtype != Py_None;
        if (known)
        {
            if (!THPDtype_Check(dtype))
                raise(PyExc_TypeError, "dtype: a torch.dtype is expected");
            type = reinterpret_cast<THPDtype*>(dtype)->scalar_type;
        }
        for (PyObject* o : tensors)
            if (o != Py_None)
            {
                require(!known || tensor(o).scalar_type() == type, "bias, residual, out and dtype: one type");
                type = tensor(o).scalar_type();
                known = true;
            }
        require(type == at::kHalf || type == at::kBFloat16, "results of fp16 or bf16");
        return type;
    }
    void fp8_activations(const Tensor& a, const Tensor& as, int& m, int& k)
    {
        matrix(a);
        m = size32(a.size(0)), k = size32(a.size(1));
        require(is(a, E4M3, {m, k}), "activations: contiguous float8_e4m3fn [M, K]");
        require(is(as, at::kFloat, {blocks128(k), m}), "scales of the activations: contiguous fp32 [ceil(K/128), M]");
    }

    // (a, a_scales, w, w_scales, bias, residual, act, out, dtype, variant)
    PyObject* fp8_gemm(Args v)
    {
        const Tensor &a = tensor(v[0]), &as = tensor(v[1]), &w = tensor(v[2]), &ws = tensor(v[3]);
        int m, k;
        fp8_activations(a, as, m, k);
        matrix(w);
        const int act = integer(v[6]), n = mxfp4_columns(w.size(0), act);
        require(is(w, E4M3, {w.size(0), k}), "weights: contiguous float8_e4m3fn [N, K]");
        require(is(ws, at::kFloat, {blocks128(n) * (act ? 2 : 1), blocks128(k)}), "scales of the weights: contiguous fp32 [ceil(N/128), ceil(K/128)], with SiLU-gate twice");
        const at::ScalarType type = fp8_result({v[7], v[5], v[4]}, v[8]);
        if (v[4] != Py_None)
            require(is(tensor(v[4]), type, {n}), "bias: contiguous [N]");
        if (v[5] != Py_None)
            require(is(tensor(v[5]), type, {m, n}), "residual: contiguous [M, N]");
        if (v[7] != Py_None)
            require(is(tensor(v[7]), type, {m, n}), "out: contiguous [M, N]");
        on_device(a, {v[1], v[2], v[3], v[4], v[5], v[7]});
        const c10::hip::HIPGuardMasqueradingAsCUDA guard(a.device());
        Owned y(output(v[7], {m, n}, type, a, "out"));
        call("nnf_fp8_gemm", nnf_fp8_gemm_variant, stream(), a.data_ptr(), as.data_ptr(), w.data_ptr(), ws.data_ptr(), y.data(),
             type == at::kHalf ? NNF_TYPE_F16 : NNF_TYPE_BF16, m, n, k, address(v[4]), address(v[5]), act, integer(v[9]));
        return y.release();
    }

    // (a, a_scales, w, w_scales, offsets, act, out, dtype, variant)
    PyObject* fp8_grouped_gemm(Args v)
    {
        const Tensor &a = tensor(v[0]), &as = tensor(v[1]), &w = tensor(v[2]), &ws = tensor(v[3]), &offsets = tensor(v[4]);
        int m, k;
        fp8_activations(a, as, m, k);
        if (w.dim() != 3)
            raise(PyExc_ValueError, "weights [experts, N, K] are expected");
        const int experts = size32(w.size(0)), act = integer(v[5]), n = mxfp4_columns(w.size(1), act);
        require(is(w, E4M3, {experts, w.size(1), k}), "weights: contiguous float8_e4m3fn [experts, N, K]");
        require(is(ws, at::kFloat, {experts, blocks128(n) * (act ? 2 : 1), blocks128(k)}),
                "scales of the weights: contiguous fp32 [experts, ceil(N/128), ceil(K/128)], with SiLU-gate twice the blocks of N");
        require(is(offsets, at::kInt, {(int64_t)experts + 1}), "offsets: contiguous int32 [experts + 1]");
        const at::ScalarType type = fp8_result({v[6]}, v[7]);
        if (v[6] != Py_None)
            require(is(tensor(v[6]), type, {m, n}), "out: contiguous [M, N]");
        on_device(a, {v[1], v[2], v[3], v[4], v[6]});
        const c10::hip::HIPGuardMasqueradingAsCUDA guard(a.device());
        Owned y(output(v[6], {m, n}, type, a, "out"));
        call("nnf_fp8_grouped_gemm", nnf_fp8_grouped_gemm_variant, stream(), a.data_ptr(), as.data_ptr(), w.data_ptr(), ws.data_ptr(), offsets.data_ptr(), y.data(),
             type == at::kHalf ? NNF_TYPE_F16 : NNF_TYPE_BF16, experts, m, n, k, act, integer(v[8]));
        return y.release();
    }

    template <PyObject* (*F)(Args), int N>
    PyObject* entry(PyObject*, Args v, Py_ssize_t n)
    {
        if (n != N)
        {
            PyErr_Format(PyExc_TypeError, "%d arguments expected, %zd given", N, n);
            return nullptr;
        }
        try
        {
            return F(v);
        }
        catch (const Raised&)
        {
        }
        catch (const std::exception& e)
        {
            PyErr_SetString(PyExc_RuntimeError, e.what());
        }
        return nullptr;
    }

    PyObject* set_error(PyObject*, PyObject* type)
    {
        Py_INCREF(type);
        Py_XDECREF(g_error);
        g_error = type;
        Py_RETURN_NONE;
    }

#define NNF_ENTRY(f, n) {#f, (PyCFunction)(void (*)(void))entry<f, n>, METH_FASTCALL, nullptr}
    PyMethodDef methods[] = {NNF_ENTRY(w4a16_gemm, 7),       NNF_ENTRY(wna16_gemm, 11),      NNF_ENTRY(w4a16_gemm_fused, 14), NNF_ENTRY(fused_mlp_w4a16, 13),
                             NNF_ENTRY(wna16_gemm_fused, 14), NNF_ENTRY(fused_mlp_wna16, 14), NNF_ENTRY(w8a8_gemm, 7),         NNF_ENTRY(w8a8_gemm_acc, 5),
                             NNF_ENTRY(elementwise, 4),       NNF_ENTRY(rms_norm, 4),         NNF_ENTRY(dequantize, 7),        NNF_ENTRY(mxfp4_quantize, 4),
                             NNF_ENTRY(mxfp4_dequantize, 3),  NNF_ENTRY(mxfp4_gemm, 10),        NNF_ENTRY(mxfp4_grouped_gemm, 9),
                             NNF_ENTRY(moe_route, 12),        NNF_ENTRY(moe_combine, 5),       NNF_ENTRY(fp8_quantize, 4),      NNF_ENTRY(fp8_quantize_weights, 3),
                             NNF_ENTRY(fp8_gemm, 10),         NNF_ENTRY(fp8_grouped_gemm, 9),  {"set_error", set_error, METH_O, nullptr},
                             {nullptr, nullptr, 0, nullptr}};
    PyModuleDef module = {PyModuleDef_HEAD_INIT, "nnf_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};
} // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_nnf_torch()
{
    return PyModule_Create(&module);
}
