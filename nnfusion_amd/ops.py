"""Thin torch-tensor front over the C ABI (device pointers + the current HIP stream).

torch is used for device memory and streams only; every computation happens in
libnnf_hip_kernels.so.  A non-zero status from the library raises NnfError (the emitted host
wrappers of the codegen path throw std::runtime_error in the same situation).
"""
import ctypes

import torch

from . import _lib


class NnfPlan(ctypes.Structure):
    """struct nnf_plan of the C header: what a kernel-selection candidate fixes about the tile GEMM, and the
    synchronisation words that make the fp16 x int4 tile GEMM a single launch."""
    _fields_ = [("tile_rows", ctypes.c_int), ("k_parts", ctypes.c_int), ("tile_cols", ctypes.c_int),
                ("sync_flags", ctypes.c_void_p), ("sync_flags_bytes", ctypes.c_size_t), ("spin_limit", ctypes.c_int)]


SYNC_FLAGS_BYTES = 64 << 10  # NNF_SYNC_FLAGS_BYTES


def sync_flags(device):
    """A zeroed buffer for nnf_plan::sync_flags (cleared once here; every call leaves it zero again)."""
    return torch.zeros(SYNC_FLAGS_BYTES, dtype=torch.uint8, device=device)


def _plan_arg(plan, sync=None, spin_limit=0):
    """None, an NnfPlan or a (tile_rows, k_parts[, tile_cols]) tuple, plus an optional sync_flags tensor
    -> (object to keep alive, pointer argument)."""
    if plan is None and sync is None:
        return None, None
    if not isinstance(plan, NnfPlan):
        t = tuple(plan) if plan is not None else (0, 0, 0)
        plan = NnfPlan(int(t[0]), int(t[1]), int(t[2]) if len(t) > 2 else 0, None, 0, 0)
    if sync is not None:
        plan.sync_flags = sync.data_ptr()
        plan.sync_flags_bytes = sync.numel() * sync.element_size()
        plan.spin_limit = int(spin_limit)
    return plan, ctypes.cast(ctypes.pointer(plan), ctypes.c_void_p)


class NnfError(RuntimeError):
    def __init__(self, status, where):
        self.status = status
        msg = _lib.kernels().nnf_status_string(status).decode()
        super().__init__(f"{where}: status {status} ({msg})")


class _Native:
    """The functions of the native front (csrc/torch_front/nnf_torch.cpp), loaded at the first use of one: they take the
    tensors and plain values in the order of the calls below, check them, allocate an output or workspace that was not
    given and call the C ABI on the current stream."""

    def __getattr__(self, name):
        module = _lib.torch_front()
        module.set_error(NnfError)
        for f in dir(module):
            if not f.startswith("_"):
                setattr(self, f, getattr(module, f))
        return getattr(module, name)


_native = _Native()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _check(status, where):
    if status != 0:
        raise NnfError(status, where)


def _ws(nbytes, device):
    # the library never allocates; the caller (here: the test/bench harness) owns the workspace
    return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=device)


def _p(t):
    return 0 if t is None else t.data_ptr()


def w4a16_gemm(a, wq, scales, group=128, zp=8, out=None, workspace=None):
    """Y[M,N] = A[M,K] . ((Wq - zp) * scales)^T ; a fp16 [M,K], wq u8 [N,K/2], scales fp16 [N,K/group]."""
    return _native.w4a16_gemm(a, wq, scales, group, zp, out, workspace)


class NnfQuant(ctypes.Structure):
    """struct nnf_quant of the C header: the block parameters of the weights."""
    _fields_ = [("bits", ctypes.c_int), ("group", ctypes.c_int), ("zero_point", ctypes.c_int),
                ("zero_points", ctypes.c_void_p)]


def _quant_arg(bits, group, zp, zero_points):
    q = NnfQuant(int(bits), int(group), int(zp), _p(zero_points))
    return q, ctypes.cast(ctypes.pointer(q), ctypes.c_void_p)


def wna16_supported(m, n, k, bits, group, zp=8):
    _, qp = _quant_arg(bits, group, zp, None)
    return bool(_lib.kernels().nnf_wna16_supported(m, n, k, qp))


def wna16_workspace_bytes(m, n, k, bits, group, zero_points=None):
    """Bytes of workspace nnf_wna16_gemm wants for this product (0: none)."""
    _, qp = _quant_arg(bits, group, 0, zero_points)
    return int(_lib.kernels().nnf_wna16_gemm_preferred_workspace_bytes(m, n, k, qp))


def wna16_gemm(a, wq, scales, bits=4, group=128, zp=8, zero_points=None, out=None, workspace=None, sync=None, spin_limit=0):
    """Y[M,N] = A[M,K] . ((Wq - z) * scales)^T with 4- or 8-bit weights (wq u8 [N, K*bits/8]), groups of 32 / 64 / 128
    and either a scalar zero point or zero_points u8 [N, ceil(K/group*bits/8)] (4-bit: two per byte, even group low).
    sync: synchronisation words (sync_flags()) for the one-launch form of the tile GEMM: nnf_wna16_gemm_planned."""
    return _native.wna16_gemm(a, wq, scales, bits, group, zp, zero_points, out, workspace, sync, spin_limit)


VARIANTS = {"auto": 0, "gemv_valu": 1, "gemv_mfma": 2, "gemm_mfma": 3, "gemv_rows": 4}


def w4a16_variant_supported(m, n, k, variant, group=128):
    return bool(_lib.kernels().nnf_w4a16_variant_supported(m, n, k, group, VARIANTS[variant]))


def w4a16_gemm_variant(a, wq, scales, variant, plan=None, group=128, zp=8, out=None, workspace=None, sync=None,
                       spin_limit=0):
    """As w4a16_gemm through one kernel variant (a key of VARIANTS) and, for the tile GEMM, a plan (tile_rows,
    k_parts); raises NnfError with status -2 when the variant cannot serve the shape."""
    lib = _lib.kernels()
    m, k = a.shape
    n = wq.shape[0]
    v = VARIANTS[variant]
    assert a.dtype == torch.float16 and wq.dtype == torch.uint8 and scales.dtype == torch.float16
    assert a.is_contiguous() and wq.is_contiguous() and scales.is_contiguous()
    if out is None:
        out = torch.empty((m, n), dtype=torch.float16, device=a.device)
    keep, plan_ptr = _plan_arg(plan, sync, spin_limit)
    if workspace is None:
        workspace = _ws(lib.nnf_w4a16_gemm_variant_workspace_bytes(m, n, k, group, v, plan_ptr), a.device)
    _check(lib.nnf_w4a16_gemm_variant(_stream(), a.data_ptr(), wq.data_ptr(), scales.data_ptr(), out.data_ptr(),
                                      m, n, k, group, zp, v, plan_ptr, workspace.data_ptr(), workspace.numel()),
           "nnf_w4a16_gemm_variant")
    return out


def w4a16_gemm_fused(a, wq, scales, group=128, zp=8, rms_gamma=None, rms_eps=1e-6, bias=None, residual=None,
                     act=0, out=None, workspace=None, variant="auto", plan=None, sync=None, spin_limit=0):
    """GEMM with the fused RMSNorm prologue / bias, residual, SiLU-gate epilogues (see the C header); variant
    "gemm_mfma" and a plan (tile_rows, k_parts) go through nnf_w4a16_gemm_fused_variant."""
    if variant == "auto" and plan is None:
        return _native.w4a16_gemm_fused(a, wq, scales, group, zp, rms_gamma, rms_eps, bias, residual, act, out, workspace, sync,
                                        spin_limit)
    lib = _lib.kernels()
    m, k = a.shape
    n = wq.shape[0] // (2 if act == 1 else 1)
    if out is None:
        out = torch.empty((m, n), dtype=torch.float16, device=a.device)
    keep, plan_ptr = _plan_arg(plan, sync, spin_limit)
    v = VARIANTS[variant]
    if workspace is None:
        need = lib.nnf_w4a16_gemm_fused_workspace_bytes(m, n, k, group, act)
        workspace = _ws(need + lib.nnf_w4a16_gemm_variant_workspace_bytes(m, wq.shape[0], k, group, v, plan_ptr), a.device)
    _check(lib.nnf_w4a16_gemm_fused_variant(_stream(), a.data_ptr(), wq.data_ptr(), scales.data_ptr(),
                                            out.data_ptr(), m, n, k, group, zp, _p(rms_gamma), float(rms_eps),
                                            _p(bias), _p(residual), int(act), v, plan_ptr, workspace.data_ptr(),
                                            workspace.numel()), "nnf_w4a16_gemm_fused_variant")
    return out


W8A8_VARIANTS = {"auto": 0, "gemv_mfma": 1, "gemm_mfma": 2, "gemv_rows": 3}


def w8a8_variant_supported(m, n, k, variant):
    return bool(_lib.kernels().nnf_w8a8_variant_supported(m, n, k, W8A8_VARIANTS[variant]))


def _w8a8_variant(a, s_tok, w, s_ch, y, acc, variant, plan, workspace, sync=None):
    lib = _lib.kernels()
    m, k = a.shape
    n = w.shape[0]
    v = W8A8_VARIANTS[variant]
    keep, plan_ptr = _plan_arg(plan, sync)
    if workspace is None:
        workspace = _ws(lib.nnf_w8a8_gemm_variant_workspace_bytes(m, n, k, v, plan_ptr), a.device)
    _check(lib.nnf_w8a8_gemm_variant(_stream(), a.data_ptr(), _p(s_tok), w.data_ptr(), _p(s_ch), _p(y), _p(acc), m, n, k,
                                     v, plan_ptr, workspace.data_ptr(), workspace.numel()), "nnf_w8a8_gemm_variant")


def w8a8_gemm(a, s_tok, w, s_ch, out=None, workspace=None, variant="auto", plan=None, sync=None):
    """Y fp16 [M,N] = fp16((float)(A . W^T) * s_tok[m] * s_ch[n]) ; a i8 [M,K], w i8 [N,K].  A variant (a key of
    W8A8_VARIANTS), a plan (tile_rows, k_parts) or `sync` (see sync_flags: with variant "gemv_rows" a few rows with a
    long K then run over two ranges of K in one launch) goes through nnf_w8a8_gemm_variant."""
    if variant == "auto" and plan is None:
        return _native.w8a8_gemm(a, s_tok, w, s_ch, out, workspace, sync)
    assert a.dtype == torch.int8 and w.dtype == torch.int8
    assert s_tok.dtype == torch.float32 and s_ch.dtype == torch.float32
    if out is None:
        out = torch.empty((a.shape[0], w.shape[0]), dtype=torch.float16, device=a.device)
    _w8a8_variant(a, s_tok, w, s_ch, out, None, variant, plan, workspace, sync)
    return out


def w8a8_gemm_acc(a, w, out=None, workspace=None, variant="auto", plan=None, sync=None):
    """acc i32 [M,N] = A . W^T, exact."""
    if variant == "auto" and plan is None:
        return _native.w8a8_gemm_acc(a, w, out, workspace, sync)
    assert a.dtype == torch.int8 and w.dtype == torch.int8
    if out is None:
        out = torch.empty((a.shape[0], w.shape[0]), dtype=torch.int32, device=a.device)
    _w8a8_variant(a, None, w, None, None, out, variant, plan, workspace, sync)
    return out


def fused_mlp_w4a16(x, gamma, wgu, sgu, wd, sd, eps=1e-6, group=128, zp=8, out=None, workspace=None, sync=None,
                    spin_limit=0, gate_up_plan=None, down_plan=None):
    """out = x + Wd . (SiLU(Wg . n) * (Wu . n)), n = RMSNorm(x, gamma, eps).  `sync` (see sync_flags) or a plan for
    either product goes through nnf_fused_mlp_w4a16_planned."""
    if gate_up_plan is None and down_plan is None:
        return _native.fused_mlp_w4a16(x, gamma, wgu, sgu, wd, sd, eps, group, zp, out, workspace, sync, spin_limit)
    lib = _lib.kernels()
    m, h = x.shape
    i = wgu.shape[0] // 2
    if out is None:
        out = torch.empty((m, h), dtype=torch.float16, device=x.device)
    keep_a, plan_a = _plan_arg(gate_up_plan, sync, spin_limit)
    keep_b, plan_b = _plan_arg(down_plan, sync, spin_limit)
    if workspace is None:
        v = VARIANTS["gemm_mfma"]
        need = lib.nnf_fused_mlp_w4a16_workspace_bytes(m, h, i, group)
        extra = (lib.nnf_w4a16_gemm_variant_workspace_bytes(m, 2 * i, h, group, v, plan_a) if gate_up_plan is not None else 0) + \
                (lib.nnf_w4a16_gemm_variant_workspace_bytes(m, h, i, group, v, plan_b) if down_plan is not None else 0)
        workspace = _ws(need + extra, x.device)
    _check(lib.nnf_fused_mlp_w4a16_planned(_stream(), x.data_ptr(), gamma.data_ptr(), float(eps), wgu.data_ptr(),
                                           sgu.data_ptr(), wd.data_ptr(), sd.data_ptr(), out.data_ptr(), m, h, i, group,
                                           zp, plan_a, plan_b, workspace.data_ptr(), workspace.numel()),
           "nnf_fused_mlp_w4a16_planned")
    return out


EW_OPS = {"add": 0, "multiply": 1, "sigmoid": 2, "swish": 3}


def elementwise(op, a, b=None, out=None):
    """y = op(a, b) over fp16 tensors (b of a's shape, or a row [cols] broadcast over a's leading axes)."""
    return _native.elementwise(EW_OPS[op], a, b, out)


def rms_norm(x, gamma, eps=1e-6, out=None):
    return _native.rms_norm(x, gamma, eps, out)


def dequantize(wq, scales, bits=4, group=128, zp=8, zero_points=None, out=None):
    """W fp16 [N, K] = (q - z) * s per block of `group` weights."""
    return _native.dequantize(wq, scales, bits, group, zp, zero_points, out)


def wna16_gemm_fused(a, wq, scales, bits=4, group=128, zp=8, zero_points=None, rms_gamma=None, rms_eps=1e-6, bias=None,
                     residual=None, act=0, out=None, workspace=None):
    """nnf_wna16_gemm_fused: the fused product for every block parameter."""
    return _native.wna16_gemm_fused(a, wq, scales, bits, group, zp, zero_points, rms_gamma, rms_eps, bias, residual, act, out,
                                    workspace)


def fused_mlp_wna16(x, gamma, wgu, sgu, wd, sd, bits=4, group=128, zp=8, zgu=None, zd=None, eps=1e-6, out=None, workspace=None):
    """The MLP block for every block parameter (zgu / zd: zero-point tensors of the two weight matrices, or None)."""
    return _native.fused_mlp_wna16(x, gamma, wgu, sgu, wd, sd, bits, group, zp, zgu, zd, eps, out, workspace)


def mxfp4_scale_bytes(k):
    """Bytes of a row of MXFP4 scale bytes: K / 32 rounded up to 16."""
    return int(_lib.kernels().nnf_mxfp4_scale_bytes(k))


def mxfp4_quantize(x, rows=None, codes=None, scales=None):
    """fp16 [source_rows, K] -> (codes u8 [rows, K/2], scales u8 [rows, mxfp4_scale_bytes(K)]): microscaled 4-bit values in blocks of
    32 along K.  rows: i32, the row of x that each quantised row is (tokens in the order of their experts; zeros where x has no
    such row), or None for every row in turn."""
    return _native.mxfp4_quantize(x, rows, codes, scales)


def mxfp4_dequantize(codes, scales, out=None):
    """The fp16 [rows, K] that MXFP4 codes and scale bytes stand for."""
    return _native.mxfp4_dequantize(codes, scales, out)


MXFP4_VARIANTS = {name: i for i, name in enumerate((
    "auto", "rows_16x16", "rows_16x32", "tile_8x32", "tile_16x32", "tile_16x32_2", "tile_16x32_4", "tile_16x64", "tile_32x64", "tile_32x128",
    "tile_64x64", "tile_64x128", "tile_64x128_deep", "tile_128x128", "tile_128x128_deep", "tile_256x256"))}


def mxfp4_variant_supported(variant, act=0):
    return bool(_lib.kernels().nnf_mxfp4_variant_supported(MXFP4_VARIANTS[variant], act))


def mxfp4_gemm_workspace_bytes(m, n, k, act=0):
    """Bytes of workspace mxfp4_gemm wants for this product (0: none)."""
    return int(_lib.kernels().nnf_mxfp4_gemm_workspace_bytes(m, n, k, act))


def mxfp4_gemm(a, a_scales, w, w_scales, bias=None, residual=None, act=0, out=None, workspace=None, variant="auto"):
    """Y fp16 [M,N] = A . W^T (+ bias + residual) of MXFP4 operands (see mxfp4_quantize), or with act=1 SiLU(gate) * up where w holds
    the gate rows, then the up rows.  fp32 sums, one rounding at the end.  out may be the residual.  variant: one kernel
    (a key of MXFP4_VARIANTS) instead of the library's choice."""
    return _native.mxfp4_gemm(a, a_scales, w, w_scales, bias, residual, act, out, workspace, MXFP4_VARIANTS[variant])


def mxfp4_grouped_gemm_workspace_bytes(experts, m, n, k, act=0):
    """Bytes of workspace mxfp4_grouped_gemm wants for this product (0: none)."""
    return int(_lib.kernels().nnf_mxfp4_grouped_gemm_workspace_bytes(experts, m, n, k, act))


def mxfp4_grouped_gemm(a, a_scales, w, w_scales, offsets, act=0, out=None, workspace=None, variant="auto"):
    """The product of a mixture's experts: rows of a sorted by expert, w u8 [experts, N, K/2] (2N rows with act=1, SiLU-gate), w_scales
    u8 [experts, N, mxfp4_scale_bytes(K)]; group e is the rows offsets[e] .. offsets[e+1] (offsets i32 [experts+1], on the device, not
    decreasing).  Rows of out that belong to no group are left as they are (undefined where out is allocated here).  The library chooses a
    kernel for all rows of a; where the groups fill little of them, name a variant for the rows there are."""
    return _native.mxfp4_grouped_gemm(a, a_scales, w, w_scales, offsets, act, out, workspace, MXFP4_VARIANTS[variant])


MOE_SCORES = {"softmax": 0, "sigmoid": 1}


def moe_route_workspace_bytes(tokens, experts, k):
    """Bytes of workspace moe_route wants (0: none)."""
    return int(_lib.kernels().nnf_moe_route_workspace_bytes(tokens, experts, k))


def moe_route(logits, k, score="softmax", bias=None, groups=1, top_groups=1, group_top=1, renormalize=True, scale=1.0, tokens=None, out=None,
              workspace=None):
    """Routing to experts: logits [tokens, experts] (fp16, bf16 or fp32) -> (weights f32 [tokens, k], experts i32 [tokens, k], rows
    i32 [tokens * k], offsets i32 [experts + 1], positions i32 [tokens, k]).  The k experts with the largest score + bias (bias f32 [experts]),
    best first, among the top_groups of `groups` groups whose group_top (1 or 2) best ones have the largest sum; ties go to the lowest index.
    weights: their scores (without the bias), divided by their sum with renormalize, times scale.  rows: the tokens sorted by expert, the `rows`
    of mxfp4_quantize and fp8_quantize; offsets: the groups of mxfp4_grouped_gemm and fp8_grouped_gemm; positions: where in that order
    a token's experts have it, for moe_combine.  A logit of -inf or NaN masks its expert (last choice, weight 0).  tokens: one i32 on the
    device, how many tokens are there (a padded batch): the others have experts and positions -1, weights 0, and their rows come last, as -1.
    out: the five results' tensors (None for one that is to be allocated)."""
    return _native.moe_route(logits, k, MOE_SCORES[score], bias, groups, top_groups, group_top, renormalize, scale, tokens, out, workspace)


def moe_combine(x, weights, positions, residual=None, out=None):
    """The experts' rows back to their tokens: out[t] = residual[t] + sum_j weights[t, j] * x[positions[t, j]]; x [rows, N] fp16 or bf16, weights and
    positions [tokens, k] as moe_route gives them.  fp32 sums, one rounding.  Positions outside x and weights of 0 add nothing.  out may be
    the residual."""
    return _native.moe_combine(x, weights, positions, residual, out)


def fp8_quantize(x, rows=None, codes=None, scales=None):
    """fp16 or bf16 [source_rows, K] -> (codes float8_e4m3fn [rows, K], scales f32 [ceil(K/128), rows]): 8-bit values with a scale for each 128 of
    a row along K, max(largest magnitude, 2^-64) / 448.  rows: i32, the row of x that each quantised row is (tokens in the order of their
    experts, as moe_route gives it; zeros where x has no such row), or None for every row in turn.  K a multiple of 16."""
    return _native.fp8_quantize(x, rows, codes, scales)


def fp8_quantize_weights(w, codes=None, scales=None):
    """fp16 or bf16 [N, K] or [matrices, N, K] -> (codes float8_e4m3fn of w's shape, scales f32 [.., ceil(N/128), ceil(K/128)]): a scale for each block of
    128 x 128.  Gate and up rows are two matrices of N rows each."""
    return _native.fp8_quantize_weights(w, codes, scales)


FP8_VARIANTS = {name: i for i, name in enumerate(("auto", "tile_16x32", "tile_16x32_2", "tile_16x32_4", "tile_32x64", "tile_64x64", "tile_64x128", "tile_128x256", "tile_256x256",
                                                       "rows_16x16", "rows_16x32"))}


def fp8_gemm(a, a_scales, w, w_scales, bias=None, residual=None, act=0, out=None, dtype=None, variant="auto"):
    """Y [M,N] = A . W^T (+ bias + residual) of block-scaled 8-bit operands: a [M,K] and a_scales [ceil(K/128), M] as fp8_quantize gives them, w [N,K] and
    w_scales [ceil(N/128), ceil(K/128)] as fp8_quantize_weights does; with act=1 SiLU(gate) * up, where w holds the gate rows, then the up
    rows, and w_scales the gate's blocks, then the up matrix's.  Sums in fp32, of products of which the 8-bit matrix instructions keep what lies within
    2^-13 of the largest of eight neighbours along K (2^-16 of the sums' root mean square for normal data); one rounding to dtype: that of out,
    residual or bias where given, else fp16 unless named.  out may be the residual.  variant: one kernel (a key of FP8_VARIANTS) instead of the library's choice."""
    return _native.fp8_gemm(a, a_scales, w, w_scales, bias, residual, act, out, dtype, FP8_VARIANTS[variant])


def fp8_grouped_gemm(a, a_scales, w, w_scales, offsets, act=0, out=None, dtype=None, variant="auto"):
    """The product of a mixture's experts: rows of a sorted by expert, w [experts, N, K] (2N rows with act=1, SiLU-gate), w_scales f32 [experts,
    ceil(N/128), ceil(K/128)] (twice the blocks with act=1); group e is the rows offsets[e] .. offsets[e+1] (offsets i32 [experts+1], on the device, not
    decreasing).  Sums as fp8_gemm's.  Rows of out that belong to no group are left as they are (undefined where out is allocated here).  The library
    chooses a kernel for all rows of a; where the groups fill little of them, name a variant for the rows there are."""
    return _native.fp8_grouped_gemm(a, a_scales, w, w_scales, offsets, act, out, dtype, FP8_VARIANTS[variant])
