"""The operators around a mixture's experts and their products in 8-bit floating point as cases that can be timed and compared: ``own`` true
makes the calls of ``nnfusion_amd.ops`` that a user makes, ``own`` false computes the same in elementary torch operations.

Routing: the experts of each token by their scores (softmax or sigmoid of the logits), chosen by score + bias among the best groups of
experts, ties to the lowest index; their weights; and the rows in the experts' order that quantising and the grouped products take.  What
decides between two experts is compared in 64 bits.  Combining: a token's row from the rows of its experts, times their weights.

The 8-bit format: E4M3 values (largest 448), 128 of them along K with one fp32 scale; for weights a block of 128 x 128 has one.  The scale is
max(largest magnitude, 2^-64) / 448, a value the fp32 quotient rounded to the nearest E4M3, ties to even.  Codes float8_e4m3fn [rows, K],
scales of activations fp32 [blocks of K, rows], of weights fp32 [blocks of N, blocks of K] (with SiLU-gate the gate's blocks, then the up
matrix's); the last block of N or K may be short.

Kinds of cases:

``route``    logits to experts, weights and the experts' order; ``spare`` tokens behind the ``tokens`` real ones (a padded batch);
``combine``  the experts' rows back to their tokens, with ``residual`` added to another row of each token (a shared expert's, or the input's);
``rows``     activations are quantised, picked by an index or not;
``weights``  a weight matrix is quantised;
``linear``   one linear layer: activations are quantised, then multiplied (bias, residual or SiLU-gate inside);
``product``  the product alone, both operands in hand (several products that share their activations quantise them once);
``experts``  the product of a mixture's experts: rows sorted by expert, ragged groups; with ``gate`` gate and up projections with SiLU-gate.

Distributions: logits N(0, 1.5), balancing biases N(0, 0.05); activations N(0, 1), one in 256 channels ten times as large, as transformer
activations have; weights N(0, 1/K); tokens go to expert e with a probability proportional to (1 + e)^-skew, the experts in an order of the
seed's.
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _route(name, tokens, experts, k, score="softmax", bias=False, groups=1, top_groups=1, group_top=1, renormalize=True, scale=1.0, type="f32", spare=0):
    return {"name": name, "kind": "route", "tokens": tokens, "experts": experts, "k": k, "score": score, "bias": bias, "groups": groups,
            "top_groups": top_groups, "group_top": group_top, "renormalize": renormalize, "scale": scale, "type": type, "spare": spare}


def _combine(name, tokens, k, n, residual=False, type="f16"):
    return {"name": name, "kind": "combine", "tokens": tokens, "k": k, "n": n, "residual": residual, "type": type}


def _pack(name, kind, m, k, tokens=0, type="f16"):
    return {"name": name, "kind": kind, "m": m, "k": k, "tokens": tokens, "type": type}


def _linear(name, m, n, k, bias=False, residual=False, gate=False, kind="linear", type="f16"):
    return {"name": name, "kind": kind, "m": m, "n": n, "k": k, "bias": bias, "residual": residual, "gate": gate, "type": type}


def _experts(name, experts, m, n, k, gate=False, skew=0.5, pad=0, type="f16"):
    return {"name": name, "kind": "experts", "experts": experts, "m": m, "n": n, "k": k, "gate": gate, "skew": skew, "pad": pad, "type": type}


def listed():
    return [
        # a single token of decoding: sigmoid scores, balancing bias, four of eight groups; the smallest call
        _route("route_m1", 1, 256, 8, "sigmoid", True, 8, 4, 2, scale=2.5),
        # an odd batch captured for 512 tokens, 333 of them real; experts in no power of two, weights as they are
        _route("route_odd", 333, 60, 4, renormalize=False, type="f16", spare=179),
        # a long prefill over many experts
        _route("route_prefill", 16384, 128, 8, type="bf16"),
        # decoding 64 tokens, six experts each, back to their rows
        _combine("combine_m64", 64, 6, 5504),
        # a long prefill, eight experts each, onto the residual
        _combine("combine_prefill", 8192, 8, 4096, residual=True, type="bf16"),
        # 1000 tokens to four experts each: the rows are quantised in the experts' order
        _pack("rows_gathered", "rows", 4000, 5504, tokens=1000),
        # a whole gate | up weight matrix of a Llama-7B layer
        _pack("weights_gate_up", "weights", 22016, 4096, type="bf16"),
        # batched decoding through the gate and up projections
        _linear("gate_up_m16", 16, 11008, 4096, gate=True, type="bf16"),
        # an odd batch, odd columns, a short last block of K and of N
        _linear("linear_odd_m45", 45, 4099, 2080, bias=True),
        # the largest dense product: a long prefill through a square layer
        _linear("prefill_m4096", 4096, 8192, 8192, kind="product", type="bf16"),
        # decoding 16 tokens, four of 32 experts each: every expert that is met streams its weights for a row or three
        _experts("experts_decode", 32, 64, 2048, 4096, gate=True),
        # a long prefill over many small experts, the row buffer longer than the tokens fill it
        _experts("experts_prefill", 64, 16000, 4096, 2048, skew=0.7, pad=384, type="bf16"),
    ]


def _log_uniform(rng, low, high):
    return math.exp(rng.uniform(math.log(low), math.log(high)))


def _width(rng, low, high):
    """Columns of a layer: usually a multiple of 128, now and then any number."""
    n = int(_log_uniform(rng, low, high))
    return max(low, n // 128 * 128) if rng.random() < 0.7 else n


def _depth(rng, low, high):
    """K: usually a multiple of 128, now and then of 16 only."""
    k = int(_log_uniform(rng, low, high))
    return max(128, k // 128 * 128) if rng.random() < 0.75 else k // 16 * 16


def _draw_route(rng):
    experts, k = int(_log_uniform(rng, 4, 513)), int(_log_uniform(rng, 1, 17))
    groups = rng.choice([g for g in (1, 1, 2, 4, 8, 16) if experts % g == 0 and experts // g >= 2])
    top_groups = rng.randint(1, groups)
    case = _route("", int(_log_uniform(rng, 1, 16385)), experts, 1, rng.choice(("softmax", "sigmoid")), rng.random() < 0.5, groups, top_groups, rng.choice((1, 2)),
                  rng.random() < 0.7, rng.choice((1.0, 2.5)), rng.choice(("f32", "f16", "bf16")), rng.choice((0, 0, 1, 100)))
    case["k"] = min(k, experts // groups * top_groups)
    return case


def draw(rng):
    """One more case of the ranges: 1 .. 16384 tokens over 4 .. 512 experts, up to 16 each; 1 .. 32768 rows quantised, matrices up to 22016 rows;
    1 .. 4096 rows of a dense layer with 64 .. 22016 columns and K = 128 .. 16384; 2 .. 128 experts with 1 .. 16384 rows in all."""
    while True:
        kind = rng.choice(("route", "route", "combine", "rows", "weights", "linear", "linear", "product", "experts", "experts", "experts"))
        type = rng.choice(("f16", "bf16"))
        if kind == "route":
            case = _draw_route(rng)
        elif kind == "combine":
            case = _combine("", int(_log_uniform(rng, 1, 8193)), rng.randint(1, 8), _width(rng, 64, 8193), rng.random() < 0.5, type)
        elif kind == "rows":
            m = int(_log_uniform(rng, 1, 32769))
            case = _pack("", kind, m, _depth(rng, 128, 16385), max(1, m // rng.choice((1, 2, 4, 8))) if rng.random() < 0.5 else 0, type)
        elif kind == "weights":
            case = _pack("", kind, _width(rng, 64, 22017), _depth(rng, 128, 16385), 0, type)
        elif kind == "experts":
            case = _experts("", int(_log_uniform(rng, 2, 129)), int(_log_uniform(rng, 1, 16385)), _width(rng, 64, 11009), _depth(rng, 128, 8193),
                            rng.random() < 0.5, rng.choice((0.0, 0.5, 1.0, 2.0)), rng.choice((0, 0, 1, 100)), type)
        else:
            gate = rng.random() < 0.3
            case = _linear("", int(_log_uniform(rng, 1, 4097)), _width(rng, 64, 11009 if gate else 22017), _depth(rng, 128, 16385),
                           not gate and rng.random() < 0.3, not gate and rng.random() < 0.3, gate, kind, type)
        del case["name"]
        w = work(case)
        if w["flops"] <= 5.4e11 and w["bytes"] <= 7.4e8 and _weight_values(case) <= 6e8:
            return case


def _weight_values(case):
    return case.get("experts", 1) * case["n"] * (2 if case["gate"] else 1) * case["k"] if "gate" in case else 0


def _shares(case):
    p = [(1.0 + e) ** -case["skew"] for e in range(case["experts"])]
    return [v / sum(p) for v in p]


def _blocks(size):
    return -(-size // 128)


def _pair(rows, k):
    """Bytes of quantised rows: a byte a value, four for a block."""
    return rows * (k + 4 * _blocks(k))


def work(case):
    """Each operand read once, each result written once."""
    kind, size = case["kind"], 4 if case["type"] == "f32" else 2
    if kind == "route":
        t, e, k = case["tokens"] + case["spare"], case["experts"], case["k"]
        # a score, a comparison or two for each expert and for each of the k; weights, experts, positions and rows of four bytes
        return {"bytes": t * (e * size + 16 * k) + 4 * (e + 1), "flops": case["tokens"] * e * (4 + k)}
    if kind == "combine":
        t, k, n = case["tokens"], case["k"], case["n"]
        return {"bytes": 2 * t * n * (k + 1 + (1 if case["residual"] else 0)) + 8 * t * k, "flops": 2 * t * k * n}
    m, k = case["m"], case["k"]
    if kind in ("rows", "weights"):
        source = min(m, case["tokens"]) if case["tokens"] else m
        scales = _blocks(k) * (m if kind == "rows" else _blocks(m)) * 4
        return {"bytes": 2 * source * k + m * k + scales + (4 * m if case["tokens"] else 0), "flops": 3 * m * k}
    n, rows = case["n"], case["n"] * (2 if case["gate"] else 1)
    matrices = 1
    if kind == "experts":
        # the experts that no row goes to are not read (expected number)
        matrices = sum(1 - (1 - p) ** m for p in _shares(case))
    total = matrices * (rows * k + 4 * _blocks(k) * _blocks(n) * (rows // n)) + m * n * 2
    # a linear layer reads 16-bit activations, writes and reads the quantised ones
    total += 2 * m * k + 2 * _pair(m, k) if kind == "linear" else _pair(m, k)
    total += (2 * n if case.get("bias") else 0) + (2 * m * n if case.get("residual") else 0) + (4 * (case["experts"] + 1) if kind == "experts" else 0)
    return {"bytes": int(total), "flops": 2 * m * rows * k}


# ---- the plain form -----------------------------------------------------------------------------------------------------------


def _order(choice, excluded=None):
    """Columns by falling value, ties by rising index; excluded ones behind all others."""
    order = torch.sort(choice, dim=1, descending=True, stable=True)[1]
    if excluded is None:
        return order
    return order.gather(1, torch.sort(excluded.gather(1, order).int(), dim=1, stable=True)[1])


def _routed(logits, bias, live, case):
    total, n = logits.shape
    k, groups = case["k"], case["groups"]
    lowest, most = -math.inf, torch.finfo(torch.float32).max
    v = torch.where(torch.isnan(logits), lowest, logits.float().clamp(max=most)).double()
    masked = v == lowest
    if case["score"] == "softmax":
        top = v.amax(1, keepdim=True)
        e = torch.exp(v - torch.where(top == lowest, 0.0, top))
        s = e / e.sum(1, keepdim=True).clamp(min=1e-300)
    else:
        s = 1 / (1 + torch.exp(-v))
    # without a bias, scores are in the order of their logits
    c = s if bias is None else s + bias.double()
    c = torch.where(masked | torch.isnan(c), lowest, c)
    choice = v if bias is None else c
    excluded = None
    if case["top_groups"] < groups:
        best = torch.sort((choice if case["group_top"] == 1 else c).view(total, groups, -1), dim=2, descending=True)[0]
        kept = _order(best[:, :, :case["group_top"]].sum(2))[:, :case["top_groups"]]
        excluded = torch.ones((total, groups), dtype=torch.bool, device=logits.device).scatter(1, kept, False).repeat_interleave(n // groups, 1)
    experts = _order(choice, excluded)[:, :k]
    w = torch.where(choice.gather(1, experts) == lowest, 0.0, s.gather(1, experts))
    if case["renormalize"]:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    there = (torch.arange(total, device=logits.device) < live).unsqueeze(1)
    weights = torch.where(there, w * case["scale"], 0.0).float()
    experts = torch.where(there, experts, -1).int()
    # the (token, slot) pairs in the order of their experts; those of tokens that are not there behind all
    flat = torch.where(experts < 0, n, experts).flatten().long()
    expert, order = torch.sort(flat, stable=True)
    rows = torch.where(expert < n, order // k, -1).int()
    positions = torch.empty_like(order).scatter_(0, order, torch.arange(total * k, device=logits.device))
    positions = torch.where(there, positions.view(total, k), -1).int()
    offsets = torch.searchsorted(expert, torch.arange(n + 1, device=logits.device)).int()
    return weights, experts, rows, offsets, positions


def _scale_of(top):
    # (a quotient by a number is a product with its rounded inverse in torch: in 32 bits the last bit would be off, and with it codes next to a tie)
    return (top.clamp(min=2.0 ** -64).double() / 448).float()


def _quantized(x, block_rows):
    """[rows, K] -> codes, scales [blocks of rows, blocks of K]; a block with an infinity or NaN: scale NaN, codes 0."""
    rows, k = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -k % 128, 0, -rows % block_rows)).view(-1, block_rows, _blocks(k), 128)
    top = v.abs().amax((1, 3))
    fine = torch.isfinite(top)
    scales = torch.where(fine, _scale_of(torch.where(fine, top, 1.0)), math.nan)
    q = torch.where(fine[:, None, :, None], v / scales[:, None, :, None], 0.0)
    return q.view(-1, _blocks(k) * 128)[:rows, :k].to(torch.float8_e4m3fn), scales


def _quantized_rows(x):
    codes, scales = _quantized(x, 1)
    return codes, scales.t().contiguous()


def _spread(scales, rows, k, block_rows):
    """Scales [blocks of rows, blocks of K] for each value."""
    return scales.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :k]


def _weight_values_of(w, scales, n):
    """The numbers that weight codes stand for; the scales' blocks start anew with the up matrix."""
    k = w.shape[1]
    parts = w.shape[0] // n
    s = scales.view(parts, _blocks(n), -1).repeat_interleave(128, 1)[:, :n].reshape(parts * n, -1)
    return w.float() * _spread(s, parts * n, k, 1)


def _product(a, w, case, bias=None, residual=None):
    y = a @ w.t()
    if case["gate"]:
        gate, up = y[:, :case["n"]], y[:, case["n"]:]
        y = gate / (1 + torch.exp(-gate)) * up
    if bias is not None:
        y = y + bias.float()
    if residual is not None:
        y = y + residual.float()
    return y.to(TYPES[case["type"]])


# ---- the cases ------------------------------------------------------------------------------------------------------------------


def _activations(gen, rows, k, type):
    x = torch.randn((rows, k), generator=gen, device="cuda")
    loud = torch.rand((k,), generator=gen, device="cuda") < 1 / 256
    return (x * torch.where(loud, 10.0, 1.0)).to(TYPES[type])


def _weights(gen, rows, k):
    return torch.randn((rows, k), generator=gen, device="cuda") / math.sqrt(k)


def _prepare_route(case, gen):
    total = case["tokens"] + case["spare"]
    logits = (1.5 * torch.randn((total, case["experts"]), generator=gen, device="cuda")).to(TYPES[case["type"]])
    bias = 0.05 * torch.randn((case["experts"],), generator=gen, device="cuda") if case["bias"] else None
    live = torch.full((1,), case["tokens"], dtype=torch.int32, device="cuda") if case["spare"] else None
    return {"case": case, "logits": logits, "bias": bias, "live": live}


def _prepare_combine(case, gen):
    t, k, n = case["tokens"], case["k"], case["n"]
    weights = torch.rand((t, k), generator=gen, device="cuda") + 0.05
    return {"case": case, "weights": weights / weights.sum(1, keepdim=True), "y": _activations(gen, t * k, n, case["type"]),
            "positions": torch.randperm(t * k, generator=gen, device="cuda").int().view(t, k),
            "residual": _activations(gen, t, n, case["type"]) if case["residual"] else None}


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if case["kind"] == "route":
        return _prepare_route(case, gen)
    if case["kind"] == "combine":
        return _prepare_combine(case, gen)
    m, k, type = case["m"], case["k"], case["type"]
    state = {"case": case}
    if case["kind"] == "weights":
        state["w"] = _weights(gen, m, k).to(TYPES[type])
        return state
    state["x"] = _activations(gen, case.get("tokens") or m + case.get("pad", 0), k, type)
    if case["kind"] == "rows":
        state["rows"] = torch.randint(0, case["tokens"], (m,), generator=gen, device="cuda", dtype=torch.int32) if case["tokens"] else None
        return state
    n, experts = case["n"], case.get("experts", 1)
    # gate and up are matrices of their own, and so is each expert's
    packed = [_quantized(_weights(gen, n, k), 128) for _ in range(experts * (2 if case["gate"] else 1))]
    state["w"], state["w_scales"] = torch.cat([p[0].view(torch.uint8) for p in packed]).view(torch.float8_e4m3fn), torch.cat([p[1] for p in packed])
    if case["kind"] != "linear":
        state["a"], state["a_scales"] = _quantized_rows(state.pop("x"))
    if case["kind"] == "experts":
        state["w"], state["w_scales"] = state["w"].view(experts, -1, k), state["w_scales"].view(experts, -1, _blocks(k))
        share = torch.tensor(_shares(case), device="cuda")[torch.randperm(experts, generator=gen, device="cuda")]
        to = torch.multinomial(share, m, replacement=True, generator=gen)
        state["sizes"] = torch.bincount(to, minlength=experts).tolist()
        ends = torch.tensor([0] + state["sizes"], dtype=torch.int32).cumsum(0)
        state["offsets"] = ends.to(torch.int32).cuda()
        # (rows behind the last group belong to nobody: whoever owns the buffer finds them as they were)
        state["out"] = torch.zeros((m + case["pad"], n), dtype=TYPES[type], device="cuda")
    else:
        state["bias"] = torch.randn((n,), generator=gen, device="cuda").to(TYPES[type]) if case["bias"] else None
        state["residual"] = torch.randn((m, n), generator=gen, device="cuda").to(TYPES[type]) if case["residual"] else None
        state["out"] = torch.empty((m, n), dtype=TYPES[type], device="cuda")
    return state


def _own(state):
    from nnfusion_amd import ops

    case = state["case"]
    act = 1 if case.get("gate") else 0
    if case["kind"] == "route":
        return ops.moe_route(state["logits"], case["k"], score=case["score"], bias=state["bias"], groups=case["groups"], top_groups=case["top_groups"],
                             group_top=case["group_top"], renormalize=case["renormalize"], scale=case["scale"], tokens=state["live"])
    if case["kind"] == "combine":
        return ops.moe_combine(state["y"], state["weights"], state["positions"], residual=state["residual"])
    if case["kind"] == "rows":
        return ops.fp8_quantize(state["x"], rows=state["rows"])
    if case["kind"] == "weights":
        return ops.fp8_quantize_weights(state["w"])
    if case["kind"] == "experts":
        return ops.fp8_grouped_gemm(state["a"], state["a_scales"], state["w"], state["w_scales"], state["offsets"], act=act, out=state["out"])
    a, a_scales = ops.fp8_quantize(state["x"]) if case["kind"] == "linear" else (state["a"], state["a_scales"])
    return ops.fp8_gemm(a, a_scales, state["w"], state["w_scales"], bias=state["bias"], residual=state["residual"], act=act, out=state["out"])


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    kind = case["kind"]
    if kind == "route":
        total = state["logits"].shape[0]
        return _routed(state["logits"], state["bias"], total if state["live"] is None else state["live"], case)
    if kind == "combine":
        w = state["weights"].unsqueeze(2)
        y = (state["y"].float()[state["positions"].long()] * w).sum(1)
        return (y if state["residual"] is None else y + state["residual"].float()).to(TYPES[case["type"]])
    if kind == "rows":
        return _quantized_rows(state["x"] if state["rows"] is None else state["x"][state["rows"]])
    if kind == "weights":
        return _quantized(state["w"], 128)
    k, n = case["k"], case["n"]
    a, a_scales = _quantized_rows(state["x"]) if kind == "linear" else (state["a"], state["a_scales"])
    a = a.float() * _spread(a_scales.t(), a.shape[0], k, 1)
    if kind == "experts":
        # (a product of its own for each expert: one batched product would take the largest group's rows for all of them)
        first = 0
        for e, size in enumerate(state["sizes"]):
            if size:
                w = _weight_values_of(state["w"][e], state["w_scales"][e], n)
                state["out"][first:first + size] = _product(a[first:first + size], w, case)
            first += size
        return state["out"]
    return _product(a, _weight_values_of(state["w"], state["w_scales"], n), case, state["bias"], state["residual"])


# ---- from the definitions, in 64 bits -------------------------------------------------------------------------------------------------


def _exact_best(values, open_, count):
    """Indices of the `count` largest of each row, one after the other: the first that reaches the row's maximum among the open ones."""
    picked, open_ = [], open_.clone()
    index = torch.arange(values.shape[1], device=values.device).expand_as(values)
    for _ in range(count):
        top = torch.where(open_, values, -math.inf).amax(1, keepdim=True)
        at = torch.where(open_ & (values >= top), index, values.shape[1]).amin(1, keepdim=True)
        picked.append(at)
        open_.scatter_(1, at, False)
    return torch.cat(picked, 1)


def _exact_route(state):
    case = state["case"]
    x = state["logits"].double()
    total, n = x.shape
    k, live = case["k"], case["tokens"]
    s = torch.softmax(x, 1) if case["score"] == "softmax" else torch.sigmoid(x)
    c = s if state["bias"] is None else s + state["bias"].double()
    open_ = torch.ones_like(x, dtype=torch.bool)
    if case["top_groups"] < case["groups"]:
        size = n // case["groups"]
        best = torch.stack([c[:, g * size:(g + 1) * size].topk(case["group_top"], 1)[0].sum(1) for g in range(case["groups"])], 1)
        kept = _exact_best(best, torch.ones_like(best, dtype=torch.bool), case["top_groups"])
        open_ = (torch.arange(n, device=x.device) // size == kept.unsqueeze(2)).any(1)
    experts = _exact_best(x if state["bias"] is None else c, open_, k)
    w = torch.gather(s, 1, experts)
    w = (w / (w.sum(1, keepdim=True) + 1e-20) if case["renormalize"] else w) * case["scale"]
    w[live:] = 0
    experts[live:] = -1
    # where a pair goes: the pairs of lower experts, and those of its own ahead of it
    hot = (experts.unsqueeze(2) == torch.arange(n, device=x.device)).view(total * k, n)
    offsets = torch.nn.functional.pad(hot.sum(0).cumsum(0), (1, 0))
    at = ((hot.int().cumsum(0) - 1 + offsets[:-1]) * hot).sum(1)
    rows = torch.full((total * k,), -1, dtype=torch.long, device=x.device)
    rows[at[:live * k]] = torch.arange(live * k, device=x.device) // k
    at[live * k:] = -1
    return w, experts.int(), rows.int(), offsets.int(), at.view(total, k).int()


def _exact_blocks(x, block_rows):
    """Values of quantised rows and scales: each value's nearest one, found from its own power of two."""
    rows, k = x.shape
    v = torch.zeros((_blocks(rows) * 128 if block_rows > 1 else rows, _blocks(k) * 128), dtype=torch.float64, device=x.device)
    v[:rows, :k] = x
    v = v.unflatten(1, (-1, 128)).unflatten(0, (-1, block_rows))
    scale = torch.clamp(v.abs().amax((1, 3)), min=2.0 ** -64) / 448
    q = (v / scale.float().double()[:, None, :, None]).float().double()
    unit = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(q / unit) * unit).flatten(2).flatten(0, 1)[:rows, :k], scale


def _exact_matrix(codes, scales, n):
    """The numbers that weight codes stand for, from their bits: sign, four bits of exponent (bias 7), three of mantissa."""
    bits = codes.view(torch.uint8).long()
    e, f = bits // 8 % 16, (bits % 8).double() / 8
    v = torch.where(e == 0, torch.ldexp(f, torch.full_like(e, -6)), torch.ldexp(1 + f, e - 7)) * (1 - 2.0 * (bits // 128))
    row = torch.arange(v.shape[0], device=v.device)
    block = row // n * _blocks(n) + row % n // 128
    return v * scales.double()[block][:, torch.arange(v.shape[1], device=v.device) // 128]


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "route":
        return _exact_route(state)
    if kind == "combine":
        out = state["residual"].double() if case["residual"] else torch.zeros((case["tokens"], case["n"]), dtype=torch.float64, device="cuda")
        for j in range(case["k"]):
            out = out + state["weights"][:, j:j + 1].double() * state["y"].index_select(0, state["positions"][:, j].long()).double()
        return out
    if kind == "rows":
        x = state["x"] if state["rows"] is None else state["x"].index_select(0, state["rows"].long())
        parts = [_exact_blocks(p, 1) for p in x.split(4096)]
        return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts]).T.contiguous()
    if kind == "weights":
        parts = [_exact_blocks(p, 128) for p in state["w"].split(4096)]
        return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])
    n = case["n"]

    def layer(a, w, w_scales):
        w = _exact_matrix(w, w_scales, n)
        y = torch.cat([torch.mm(a, p.T) for p in w.split(4096)], 1)
        return y[:, :n] * torch.sigmoid(y[:, :n]) * y[:, n:] if case["gate"] else y

    if kind == "linear":
        codes, scales = _exact_blocks(state["x"], 1)
        a = codes * scales.float().double().repeat_interleave(128, 1)[:, :case["k"]]
    else:
        a = _exact_matrix(state["a"], state["a_scales"].T, 1)
    if kind == "experts":
        out, at = state["out"].double(), state["offsets"].tolist()
        for e in range(case["experts"]):
            if at[e + 1] > at[e]:
                out[at[e]:at[e + 1]] = layer(a[at[e]:at[e + 1]], state["w"][e], state["w_scales"][e])
        return out
    y = layer(a, state["w"], state["w_scales"])
    for more in (state["bias"], state["residual"]):
        if more is not None:
            y = y + more.double()
    return y
