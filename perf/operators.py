"""The operators on microscaled 4-bit numbers (MXFP4) as cases that can be timed and compared: ``own`` true makes the calls of
``nnfusion_amd.ops`` that a user makes, ``own`` false computes the same in elementary torch operations.

The format: blocks of 32 values along K share one power of two, ``2^(scale byte - 127)`` (byte 255: the block is NaN); a value is
one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign, four bits, two to a byte with the even k in the low nibble.  Codes are u8 [rows, K/2],
scale bytes u8 [rows, stride] with the stride K/32 rounded up to 16.  Quantising takes floor(log2(largest magnitude)) - 2 as
the exponent of a block, rounds to the nearest value (ties to the even code) and saturates at 6.

Kinds of cases:

``pack``     fp16 rows are quantised and read back (weights packed and looked at, activations on their way through a cache); with
             ``gather`` the rows are picked by an index, as the rows of tokens sorted by expert are;
``linear``   one linear layer: fp16 activations are quantised, then multiplied with MXFP4 weights (bias, residual or SiLU-gate inside);
``product``  the product alone, both operands in hand (several products that share their activations quantise them once);
``experts``  the product of a mixture's experts: rows sorted by expert, ragged groups, one weight matrix per expert; with
             ``gate`` the experts' gate and up projections with SiLU-gate.

Distributions: activations N(0, 1), one in 256 channels ten times as large, as transformer activations have; weights
N(0, 1/K); tokens go to expert e with a probability proportional to (1 + e)^-skew, the experts in an order of the seed's.
"""
import math

import torch

own = False

TABLE = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _pack(name, m, k, tokens=0):
    return {"name": name, "kind": "pack", "m": m, "k": k, "gather": tokens > 0, "tokens": tokens}


def _linear(name, m, n, k, bias=False, residual=False, gate=False, kind="linear", keep=True):
    return {"name": name, "kind": kind, "m": m, "n": n, "k": k, "bias": bias, "residual": residual, "gate": gate, "keep": keep}


def _experts(name, experts, m, n, k, gate=False, skew=0.5, pad=0, keep=True):
    return {"name": name, "kind": "experts", "experts": experts, "m": m, "n": n, "k": k, "gate": gate, "skew": skew, "pad": pad, "keep": keep}


def listed():
    return [
        # one token's activations: the smallest call
        _pack("pack_m1", 1, 4096),
        # a whole gate | up weight matrix of a Llama-7B layer is packed and read back
        _pack("pack_weights", 22016, 4096),
        # 1000 tokens to four experts each: the rows are quantised in the experts' order
        _pack("pack_gathered", 4000, 5504, tokens=1000),
        # one token through one square layer
        _linear("linear_m1", 1, 4096, 4096),
        # batched decoding through the gate and up projections
        _linear("gate_up_m16", 16, 11008, 4096, gate=True),
        # an odd batch, odd columns, K an odd multiple of a block, plain calls
        _linear("linear_odd_m45", 45, 4099, 2080, bias=True, keep=False),
        # a chunk of a prefill through the down projection, residual added
        _linear("down_m256", 256, 4096, 11008, residual=True),
        # the largest dense product: a long prefill through a square layer
        _linear("prefill_m4096", 4096, 8192, 8192, kind="product"),
        # decoding 16 tokens, four of 32 experts each: every expert that is met streams its weights for a row or three
        _experts("experts_decode", 32, 64, 2048, 4096, gate=True),
        # 512 tokens, two of eight large experts each
        _experts("experts_m1024", 8, 1024, 11008, 4096, gate=True),
        # the experts' down projection of an odd batch: odd columns and K, experts without a row, plain call
        _experts("experts_odd", 60, 333, 2050, 1376, skew=1.5, keep=False),
        # a long prefill over many small experts, the row buffer longer than the tokens fill it
        _experts("experts_prefill", 64, 16000, 4096, 2048, skew=0.7, pad=384),
    ]


def _log_uniform(rng, low, high):
    return math.exp(rng.uniform(math.log(low), math.log(high)))


def _width(rng, low, high):
    """Columns of a layer: usually a multiple of 64, now and then any number."""
    n = int(_log_uniform(rng, low, high))
    return max(low, n // 64 * 64) if rng.random() < 0.75 else n


def _depth(rng, low, high):
    """K: usually a multiple of 128, now and then any number of blocks."""
    k = int(_log_uniform(rng, low, high))
    return max(128, k // 128 * 128) if rng.random() < 0.75 else k // 32 * 32


def draw(rng):
    """One more case of the ranges: 1 .. 4096 rows of a dense layer with 64 .. 22016 columns and K = 128 .. 16384; 2 .. 128 experts with
    1 .. 16384 rows in all; 1 .. 32768 rows packed."""
    while True:
        kind = rng.choice(("pack", "linear", "linear", "linear", "product", "experts", "experts", "experts"))
        if kind == "pack":
            m, gather = int(_log_uniform(rng, 1, 32769)), rng.random() < 0.4
            case = {"kind": kind, "m": m, "k": _depth(rng, 128, 16385), "gather": gather, "tokens": max(1, m // rng.choice((1, 2, 4, 8))) if gather else 0}
        elif kind == "experts":
            case = {"kind": kind, "experts": int(_log_uniform(rng, 2, 129)), "m": int(_log_uniform(rng, 1, 16385)), "n": _width(rng, 64, 11009),
                    "k": _depth(rng, 128, 8193), "gate": rng.random() < 0.5, "skew": rng.choice((0.0, 0.5, 1.0, 2.0)),
                    "pad": rng.choice((0, 0, 1, 100)), "keep": rng.random() < 0.7}
        else:
            gate = rng.random() < 0.3
            case = {"kind": kind, "m": int(_log_uniform(rng, 1, 4097)), "n": _width(rng, 64, 11009 if gate else 22017), "k": _depth(rng, 128, 16385),
                    "bias": not gate and rng.random() < 0.3, "residual": not gate and rng.random() < 0.3, "gate": gate, "keep": rng.random() < 0.7}
        w = work(case)
        if w["flops"] <= 5.4e11 and w["bytes"] <= 4.1e8 and _weight_values(case) <= 6e8:
            return case


def _weight_values(case):
    return 0 if case["kind"] == "pack" else case.get("experts", 1) * case["n"] * (2 if case["gate"] else 1) * case["k"]


def _shares(case):
    p = [(1.0 + e) ** -case["skew"] for e in range(case["experts"])]
    return [v / sum(p) for v in p]


def work(case):
    """Each operand read once, each result written once: 4 bits and a 32nd of a byte per MXFP4 value, 2 bytes per fp16 value."""
    m, k, packed = case["m"], case["k"], case["k"] / 2 + case["k"] / 32
    if case["kind"] == "pack":
        # quantised and read back: read fp16, write and read MXFP4, write fp16
        source = min(m, case["tokens"]) if case["gather"] else m
        return {"bytes": int(source * k * 2 + 2 * m * packed + m * k * 2 + (4 * m if case["gather"] else 0)), "flops": 3 * m * k}
    n, rows = case["n"], case["n"] * (2 if case["gate"] else 1)
    matrices = 1
    if case["kind"] == "experts":
        # the experts that no row goes to are not read (expected number)
        matrices = sum(1 - (1 - p) ** m for p in _shares(case))
    total = matrices * rows * packed + m * n * 2
    # a linear layer reads fp16 activations, writes and reads the quantised ones
    total += m * (k * 2 + 2 * packed) if case["kind"] == "linear" else m * packed
    total += (2 * n if case.get("bias") else 0) + (2 * m * n if case.get("residual") else 0) + (4 * (case["experts"] + 1) if case["kind"] == "experts" else 0)
    return {"bytes": int(total), "flops": 2 * m * rows * k}


def _stride(k):
    return (k // 32 + 15) // 16 * 16


def _quantize(x):
    """fp16 [rows, K] -> (codes, scale bytes): comparisons and products with powers of two, exact in 32 bits."""
    rows, k = x.shape
    blocks = x.float().view(rows, k // 32, 32)
    top = blocks.abs().amax(2)
    exponent = torch.frexp(top)[1] - 3  # top = f * 2^e with f in [0.5, 1)
    byte = torch.where(top == 0, torch.full_like(exponent, 127), exponent + 127)
    byte = torch.where(torch.isfinite(top), byte, torch.full_like(byte, 255))
    v = blocks * torch.exp2((127 - byte).float()).unsqueeze(2)
    a = v.abs()
    code = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte() + (a >= 3.5).byte() + (a > 5).byte()
            + 8 * (v < 0).byte()).view(rows, k // 2, 2)
    scales = torch.full((rows, _stride(k)), 127, dtype=torch.uint8, device=x.device)
    scales[:, :k // 32] = byte.to(torch.uint8)
    return code[:, :, 0] | code[:, :, 1] << 4, scales


def _values(codes, scales):
    """The numbers that codes [rows, K/2] and scale bytes stand for, in 32 bits."""
    rows, half = codes.shape
    table = torch.tensor(TABLE + tuple(-t for t in TABLE), device=codes.device)
    v = table[torch.stack((codes & 15, codes >> 4), 2).view(rows, -1, 32).int()]
    byte = scales[:, :half // 16].float()
    power = torch.where(byte == 255, torch.full_like(byte, math.nan), torch.exp2(byte - 127))
    return (v * power.unsqueeze(2)).view(rows, half * 2)


def _product(a, w, case, bias=None, residual=None):
    y = a @ w.t()
    if case["gate"]:
        gate, up = y[:, :case["n"]], y[:, case["n"]:]
        y = gate / (1 + torch.exp(-gate)) * up
    if bias is not None:
        y = y + bias.float()
    if residual is not None:
        y = y + residual.float()
    return y.half()


def _activations(gen, rows, k):
    x = torch.randn((rows, k), generator=gen, device="cuda")
    loud = torch.rand((k,), generator=gen, device="cuda") < 1 / 256
    return (x * torch.where(loud, 10.0, 1.0)).half()


def _weights(gen, rows, k):
    """A quantised matrix, made in pieces: 16 bits for all of a mixture's experts at once would be large."""
    codes, scales = [], []
    for first in range(0, rows, 16384):
        c, s = _quantize((torch.randn((min(16384, rows - first), k), generator=gen, device="cuda") / math.sqrt(k)).half())
        codes.append(c)
        scales.append(s)
    return torch.cat(codes), torch.cat(scales)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    m, k = case["m"], case["k"]
    state = {"case": case, "out": None, "workspace": None, "rows": None}
    if case["kind"] == "pack":
        state["x"] = _activations(gen, case["tokens"] if case["gather"] else m, k)
        if case["gather"]:
            state["rows"] = torch.randint(0, case["tokens"], (m,), generator=gen, device="cuda", dtype=torch.int32)
        state["codes"] = torch.empty((m, k // 2), dtype=torch.uint8, device="cuda")
        state["scales"] = torch.empty((m, _stride(k)), dtype=torch.uint8, device="cuda")
        state["out"] = torch.empty((m, k), dtype=torch.float16, device="cuda")
        return state
    n, experts, pad = case["n"], case.get("experts", 1), case.get("pad", 0)
    rows = n * (2 if case["gate"] else 1)
    x = _activations(gen, m + pad, k)
    state["w"], state["w_scales"] = _weights(gen, experts * rows, k)
    if case["kind"] == "linear":
        state["x"] = x
    else:
        state["a"], state["a_scales"] = _quantize(x)
    if case["kind"] == "experts":
        share = torch.tensor(_shares(case), device="cuda")[torch.randperm(experts, generator=gen, device="cuda")]
        to = torch.multinomial(share, m, replacement=True, generator=gen)
        state["sizes"] = torch.bincount(to, minlength=experts).tolist()
        ends = torch.tensor([0] + state["sizes"], dtype=torch.int32).cumsum(0)
        state["offsets"] = ends.to(torch.int32).cuda()
        state["w"], state["w_scales"] = state["w"].view(experts, rows, -1), state["w_scales"].view(experts, rows, -1)
        # (rows behind the last group belong to nobody: whoever owns the buffer finds them as they were)
        state["out"] = torch.zeros((m + pad, n), dtype=torch.float16, device="cuda")
    else:
        state["bias"] = torch.randn((n,), generator=gen, device="cuda").half() if case["bias"] else None
        state["residual"] = torch.randn((m, n), generator=gen, device="cuda").half() if case["residual"] else None
        if case["keep"]:
            state["out"] = torch.empty((m, n), dtype=torch.float16, device="cuda")
    if own and case["keep"]:
        from nnfusion_amd import ops

        act = 1 if case["gate"] else 0
        need = (ops.mxfp4_grouped_gemm_workspace_bytes(experts, m + pad, n, k, act) if case["kind"] == "experts"
                else ops.mxfp4_gemm_workspace_bytes(m, n, k, act))
        state["workspace"] = torch.empty((max(need, 16),), dtype=torch.uint8, device="cuda")
        if case["kind"] == "linear":
            state["codes"] = torch.empty((m, k // 2), dtype=torch.uint8, device="cuda")
            state["scales"] = torch.empty((m, _stride(k)), dtype=torch.uint8, device="cuda")
    return state


def _own(state):
    from nnfusion_amd import ops

    case = state["case"]
    act = 1 if case.get("gate") else 0
    if case["kind"] == "pack":
        codes, scales = ops.mxfp4_quantize(state["x"], rows=state["rows"], codes=state["codes"], scales=state["scales"])
        return ops.mxfp4_dequantize(codes, scales, out=state["out"])
    if case["kind"] == "experts":
        return ops.mxfp4_grouped_gemm(state["a"], state["a_scales"], state["w"], state["w_scales"], state["offsets"], act=act, out=state["out"],
                                      workspace=state["workspace"])
    if case["kind"] == "linear":
        a, a_scales = ops.mxfp4_quantize(state["x"], codes=state.get("codes"), scales=state.get("scales"))
    else:
        a, a_scales = state["a"], state["a_scales"]
    return ops.mxfp4_gemm(a, a_scales, state["w"], state["w_scales"], bias=state["bias"], residual=state["residual"], act=act, out=state["out"],
                          workspace=state["workspace"])


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    if case["kind"] == "pack":
        x = state["x"] if state["rows"] is None else state["x"][state["rows"]]
        return _values(*_quantize(x)).half()
    if case["kind"] == "experts":
        first = 0
        for e, size in enumerate(state["sizes"]):
            if size:
                a = _values(state["a"][first:first + size], state["a_scales"][first:first + size])
                state["out"][first:first + size] = _product(a, _values(state["w"][e], state["w_scales"][e]), case)
            first += size
        return state["out"]
    a = _quantize(state["x"]) if case["kind"] == "linear" else (state["a"], state["a_scales"])
    return _product(_values(*a), _values(state["w"], state["w_scales"]), case, state["bias"], state["residual"])


def _exact_matrix(codes, scales):
    """From the format's definition, value by value: sign, two bits of exponent (bias 1), one bit of mantissa, in 64 bits."""
    nibble = torch.stack((codes % 16, codes // 16), -1).flatten(-2).long()
    e, f = nibble // 2 % 4, (nibble % 2).double()
    magnitude = torch.where(e == 0, f / 2, torch.ldexp(1 + f / 2, e - 1))
    value = torch.where(nibble >= 8, -magnitude, magnitude)
    byte = scales.long().repeat_interleave(32, -1)[..., :value.shape[-1]]
    return torch.where(byte == 255, torch.full_like(value, math.nan), torch.ldexp(value, byte - 127))


def _exact_rounded(x):
    """The values that quantised fp16 rows stand for: the nearest representable one, found from the distance to each."""
    blocks = x.double().unflatten(1, (-1, 32))
    top = blocks.abs().amax(2, keepdim=True)
    unit = torch.exp2(torch.floor(torch.log2(torch.where(top == 0, torch.ones_like(top), top))) - 2)
    # ties go to the code whose last bit is zero: those are looked at first
    order = torch.tensor([0.0, 1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0], device=x.device, dtype=torch.float64)
    best, found = torch.full_like(blocks, math.inf), torch.zeros_like(blocks)
    for v in order:
        away = (blocks.abs() / unit - v).abs()
        found = torch.where(away < best, v, found)
        best = torch.minimum(best, away)
    value = torch.copysign(found * unit, blocks)
    return torch.where(torch.isfinite(top), value, torch.full_like(value, math.nan)).flatten(1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "pack":
        x = state["x"] if state["rows"] is None else state["x"].index_select(0, state["rows"].long())
        return torch.cat([_exact_rounded(piece) for piece in x.split(4096)])
    n = case["n"]

    def layer(a, w, w_scales):
        y = torch.cat([torch.mm(a, _exact_matrix(w[i:i + 4096], w_scales[i:i + 4096]).T) for i in range(0, w.shape[0], 4096)], 1)
        return y[:, :n] * torch.sigmoid(y[:, :n]) * y[:, n:] if case["gate"] else y

    if case["kind"] == "experts":
        a, out = _exact_matrix(state["a"], state["a_scales"]), state["out"].double()
        at = state["offsets"].tolist()
        for e in range(case["experts"]):
            if at[e + 1] > at[e]:
                out[at[e]:at[e + 1]] = layer(a[at[e]:at[e + 1]], state["w"][e], state["w_scales"][e])
        return out
    a = _exact_rounded(state["x"]) if case["kind"] == "linear" else _exact_matrix(state["a"], state["a_scales"])
    y = layer(a, state["w"], state["w_scales"])
    for more in (state["bias"], state["residual"]):
        if more is not None:
            y = y + more.double()
    return y
