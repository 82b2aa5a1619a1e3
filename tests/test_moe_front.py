"""What the calls of routing and combining refuse, on host tensors and at the C entry points: nothing here reaches a kernel."""
import ctypes

import pytest
import torch

from nnfusion_amd import _lib, ops

INVALID, UNSUPPORTED, TOO_SMALL, NO_DEVICE = -1, -2, -3, -4


class Routing(ctypes.Structure):
    _fields_ = [(f, ctypes.c_int) for f in ("k", "score", "groups", "top_groups", "group_top", "renormalize")] + [("scale", ctypes.c_float)]


def _at(i):
    """Addresses of made-up device buffers, far apart."""
    return (i + 1) << 33


def _route(tokens=8, E=64, workspace_bytes=1 << 20, type=2, skip=None, at=None, **routing):
    fields = {"k": 4, "score": 0, "groups": 1, "top_groups": 1, "group_top": 1, "renormalize": 1, "scale": 1.0, **routing}
    p = {name: _at(i) for i, name in enumerate(("logits", "bias", "live", "weights", "experts", "rows", "offsets", "positions", "workspace"))}
    p.update(at or {})
    if skip:
        p[skip] = None
    r = Routing(**fields)
    return _lib.kernels().nnf_moe_route(None, p["logits"], type, p["bias"], p["live"], ctypes.cast(ctypes.pointer(r), ctypes.c_void_p), p["weights"], p["experts"],
                                        p["rows"], p["offsets"], p["positions"], tokens, E, p["workspace"], workspace_bytes)


def _no_device():
    if torch.cuda.is_available():
        pytest.skip("made-up addresses: where there is a device, a call that is let through would run")


def test_routing_refuses_at_the_c_entry():
    _no_device()
    assert _route() == NO_DEVICE
    for skip in ("bias", "live", "workspace"):
        assert _route(skip=skip) == NO_DEVICE
    for skip in ("logits", "weights", "experts", "rows", "offsets", "positions"):
        assert _route(skip=skip) == INVALID
    assert _lib.kernels().nnf_moe_route(None, *[_at(0)] * 1, 2, None, None, None, _at(1), _at(2), _at(3), _at(4), _at(5), 8, 64, None, 0) == INVALID
    for bad in ({"tokens": 0}, {"tokens": -1}, {"E": 0}, {"k": 0}, {"k": -3}, {"type": 3}, {"type": -1}, {"score": 2}, {"score": -1}):
        assert _route(**bad) == INVALID, bad
    for bad in ({"E": 1025}, {"k": 17}, {"k": 65}, {"E": 8, "k": 9}, {"groups": 0}, {"groups": 17}, {"groups": 3}, {"groups": 4, "top_groups": 0},
                {"groups": 4, "top_groups": 5}, {"group_top": 0}, {"group_top": 3}, {"E": 4, "groups": 4, "top_groups": 4, "group_top": 2},
                {"E": 16, "groups": 8, "top_groups": 1, "k": 3}, {"tokens": (1 << 21) + 1}, {"tokens": 2147483647, "k": 16}):
        assert _route(**bad) == UNSUPPORTED, bad
    for good in ({"E": 1024, "k": 16}, {"E": 16, "groups": 8, "top_groups": 2, "k": 4, "group_top": 2}, {"tokens": 1 << 21, "workspace_bytes": 1 << 30}, {"E": 1, "k": 1}):
        assert _route(**good) == NO_DEVICE, good


def test_routing_wants_its_workspace():
    _no_device()
    assert ops.moe_route_workspace_bytes(1, 256, 8) == 0 and ops.moe_route_workspace_bytes(0, 256, 8) == 0
    need = ops.moe_route_workspace_bytes(1000, 256, 8)
    assert need > 0
    assert _route(tokens=1000, E=256, workspace_bytes=need) == NO_DEVICE
    assert _route(tokens=1000, E=256, workspace_bytes=need - 1) == TOO_SMALL
    assert _route(tokens=1000, E=256, skip="workspace") == TOO_SMALL


def test_routing_refuses_memory_that_overlaps_or_is_off():
    _no_device()
    names = ("logits", "bias", "live", "weights", "experts", "rows", "offsets", "positions", "workspace")
    for i, a in enumerate(names):
        for j, b in enumerate(names[:i]):
            status = _route(tokens=1000, at={a: _at(j)})
            assert status == (NO_DEVICE if i < 3 else INVALID), (a, b)
    for a in names:
        assert _route(at={a: _at(names.index(a)) + 1}) == INVALID, a
    assert _route(type=1, at={"logits": _at(0) + 2}) == NO_DEVICE and _route(type=2, at={"logits": _at(0) + 2}) == INVALID


def test_combining_refuses_at_the_c_entry():
    _no_device()

    def call(type=0, tokens=8, rows=32, k=4, n=256, **at):
        p = {"x": _at(0), "weights": _at(1), "positions": _at(2), "residual": _at(3), "y": _at(4), **at}
        return _lib.kernels().nnf_moe_combine(None, p["x"], p["weights"], p["positions"], p["residual"], p["y"], type, tokens, rows, k, n)

    assert call() == NO_DEVICE and call(residual=None) == NO_DEVICE and call(residual=_at(4)) == NO_DEVICE and call(type=1, x=_at(0) + 2) == NO_DEVICE
    for bad in ({"x": None}, {"weights": None}, {"positions": None}, {"y": None}, {"type": 2}, {"type": -1}, {"tokens": 0}, {"rows": 0}, {"k": 0}, {"n": 0},
                {"x": _at(0) + 1}, {"weights": _at(1) + 2}, {"positions": _at(2) + 2}, {"residual": _at(3) + 1}, {"y": _at(4) + 1}, {"y": _at(0)}, {"y": _at(1)}, {"y": _at(2)},
                {"residual": _at(4) + 16}):
        assert call(**bad) == INVALID, bad
    for bad in ({"k": 17}, {"tokens": 1 << 25, "n": 513}, {"tokens": 2147483647, "n": 1}):
        assert call(**bad) == UNSUPPORTED, bad


def test_routing_refuses_tensors_it_would_misread():
    x = torch.zeros((4, 8))
    for what, kw in {
        "double logits": {"logits": x.double()}, "int logits": {"logits": x.int()}, "strided logits": {"logits": x.t().contiguous().t()},
        "bias of another length": {"bias": torch.zeros(7)}, "half bias": {"bias": torch.zeros(8).half()}, "strided bias": {"bias": torch.zeros(16)[::2]},
        "int64 tokens": {"tokens": torch.tensor([3])}, "two tokens": {"tokens": torch.zeros(2, dtype=torch.int32)}, "out of four": {"out": (None,) * 4},
        "out as a list": {"out": [None] * 5}, "weights of another k": {"out": (torch.zeros((4, 3)), None, None, None, None)},
        "int64 experts": {"out": (None, torch.zeros((4, 2), dtype=torch.long), None, None, None)},
        "rows of a matrix": {"out": (None, None, torch.zeros((4, 2), dtype=torch.int32), None, None)},
        "offsets without the end": {"out": (None, None, None, torch.zeros(8, dtype=torch.int32), None)},
        "float positions": {"out": (None, None, None, None, torch.zeros((4, 2)))}, "workspace of words": {"workspace": torch.zeros(64, dtype=torch.int32)},
        "no expert": {"k": 0}, "fewer than none": {"k": -1}, "more than there are": {"k": 9}, "results of terabytes": {"k": 2**31 - 1},
        "host tensors": {},
    }.items():
        with pytest.raises(AssertionError):
            ops.moe_route(**{"logits": x, "k": 2, **kw})
            pytest.fail(what)
    for kw, error in (({"logits": x[0]}, ValueError), ({"logits": None}, TypeError), ({"k": 2.5}, TypeError), ({"k": None}, TypeError), ({"score": "tanh"}, KeyError),
                      ({"bias": [0.0] * 8}, TypeError), ({"tokens": 3}, TypeError), ({"scale": "1"}, TypeError)):
        with pytest.raises(error):
            ops.moe_route(**{"logits": x, "k": 2, **kw})


def test_combining_refuses_tensors_it_would_misread():
    x, w, p = torch.zeros((8, 16)).half(), torch.zeros((4, 2)), torch.zeros((4, 2), dtype=torch.int32)
    for what, kw in {
        "fp32 rows": {"x": x.float()}, "strided rows": {"x": torch.cat([x, x], 1)[:, ::2]}, "half weights": {"weights": w.half()}, "positions of another shape": {"positions": p[:3]},
        "int64 positions": {"positions": p.long()}, "residual of another type": {"residual": torch.zeros((4, 16)).bfloat16()}, "residual of other rows": {"residual": x[:3]},
        "out of another type": {"out": torch.zeros((4, 16))}, "host tensors": {},
    }.items():
        with pytest.raises(AssertionError):
            ops.moe_combine(**{"x": x, "weights": w, "positions": p, **kw})
            pytest.fail(what)
    for kw, error in (({"x": x[0]}, ValueError), ({"weights": w[0]}, ValueError), ({"x": None}, TypeError), ({"positions": [[0, 1]]}, TypeError)):
        with pytest.raises(error):
            ops.moe_combine(**{"x": x, "weights": w, "positions": p, **kw})
