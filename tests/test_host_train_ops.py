"""What the training operators and their C entry points refuse before any CUDA call (no GPU).

The wrappers look at the device last: a call on host tensors that is right in every other way is refused for that alone."""
import ctypes as C

import pytest
import torch

from basedxl_b200 import _lib, ops

HOST = "expected tensors of the current CUDA device, got cpu"


def _refused(call, **kw):
    with pytest.raises(ValueError) as e:
        call(**kw)
    return str(e.value)


def _z(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize(
    "kw",
    [
        {"x": _z(5, 8, dtype=torch.float64)},
        {"x": _z(5, 8, dtype=torch.int32)},
        {"x": _z(5, 0)},
        {"x": torch.zeros((), dtype=torch.float16)},
        {"weight": _z(7)},
        {"weight": _z(1, 8)},
        {"weight": _z(16)[::2]},
        {"weight": _z(8, dtype=torch.bfloat16)},
        {"bias": _z(9)},
        {"bias": _z(8, dtype=torch.float32)},        # not the weight's type
        {"out": _z(5, 9)},
        {"out": _z(8, 5).t()},
        {"out": _z(5, 8, dtype=torch.float32)},
    ],
)
def test_layernorm_fwd_refuses(kw):
    good = {"x": _z(5, 8), "weight": _z(8), "bias": _z(8)}
    assert HOST in _refused(ops.layernorm_fwd, **good)
    assert HOST not in _refused(ops.layernorm_fwd, **{**good, **kw})


@pytest.mark.parametrize(
    "kw",
    [
        {"dy": _z(5, 9)},
        {"dy": _z(8)},
        {"dy": _z(5, 8, dtype=torch.float32)},
        {"mean": _z(4, dtype=torch.float32)},
        {"mean": _z(5)},
        {"rstd": _z(10, dtype=torch.float32)[::2]},
        {"rstd": _z(5, 1, dtype=torch.float32)},
        {"weight": _z(5)},
        {"weight": _z(8, dtype=torch.bfloat16)},
    ],
)
def test_layernorm_bwd_refuses(kw):
    good = {"dy": _z(5, 8), "x": _z(5, 8), "mean": _z(5, dtype=torch.float32), "rstd": _z(5, dtype=torch.float32), "weight": _z(8)}
    assert HOST in _refused(ops.layernorm_bwd, **good)
    assert HOST not in _refused(ops.layernorm_bwd, **{**good, **kw})


@pytest.mark.parametrize(
    "kw",
    [
        {"x": _z(5, 8, dtype=torch.float32), "weight": _z(6, 8, dtype=torch.float32)},
        {"x": _z(5, 8, dtype=torch.bfloat16)},
        {"x": _z(5, 9)},
        {"weight": _z(8)},
        {"weight": _z(0, 8)},
        {"weight": _z(1, 6, 8)},
        {"bias": _z(5)},
        {"bias": _z(1, 6)},
        {"bias": _z(12)[::2]},
        {"bias": _z(6, dtype=torch.float32)},
        {"residual": _z(6)},
        {"residual": _z(5, 6, dtype=torch.float32)},
        {"activation": "swish"},
        {"activation": 3},
        {"out": _z(5, 7)},
        {"out": _z(6, 5).t()},
        {"out": _z(5, 6, dtype=torch.float32)},
    ],
)
def test_linear_act_refuses(kw):
    good = {"x": _z(5, 8), "weight": _z(6, 8), "bias": _z(6), "residual": _z(5, 6), "activation": "silu"}
    assert HOST in _refused(ops.linear_act, **good)
    assert HOST not in _refused(ops.linear_act, **{**good, **kw})


def test_results_over_inputs_are_refused():
    """Other rows of an input are still read while a result is written; in place is where a row depends on itself alone."""
    buf = _z(48)
    x, shifted = buf[:40].view(5, 8), buf[8:].view(5, 8)
    assert "out overlaps x" in _refused(ops.layernorm_fwd, x=x, out=shifted)
    wide = _z(5, 16)
    assert "out overlaps x" in _refused(ops.layernorm_fwd, x=wide[:, :8], out=wide.view(-1)[:40].view(5, 8))
    assert "out overlaps weight" in _refused(ops.layernorm_fwd, x=_z(5, 8), weight=buf[:8], out=x)
    assert "out overlaps bias" in _refused(ops.layernorm_fwd, x=_z(5, 8), bias=buf[32:40], out=x)
    assert HOST in _refused(ops.layernorm_fwd, x=x, out=x)
    assert HOST in _refused(ops.layernorm_fwd, x=x, weight=buf[40:], out=x)
    w = _z(8, 8)
    assert "out overlaps x" in _refused(ops.linear_act, x=x, weight=w, out=x)
    assert "out overlaps weight" in _refused(ops.linear_act, x=_z(8, 8), weight=w, out=w)
    assert "out overlaps bias" in _refused(ops.linear_act, x=_z(5, 8), weight=w, bias=buf[:8], out=x)
    assert "out overlaps residual" in _refused(ops.linear_act, x=_z(5, 8), weight=w, residual=x, out=shifted)
    assert HOST in _refused(ops.linear_act, x=_z(5, 8), weight=w, residual=x, out=x)


@pytest.mark.parametrize(
    "kw",
    [
        {"pre": None},
        {"pre": _z(5, 7)},
        {"pre": _z(5, 6, dtype=torch.float32)},
        {"dy": _z(5, 8)},
        {"dy": _z(5, 6, dtype=torch.bfloat16)},
        {"x": _z(4, 8)},
        {"activation": "tanh"},
    ],
)
def test_linear_act_bwd_refuses(kw):
    good = {"dy": _z(5, 6), "x": _z(5, 8), "weight": _z(6, 8), "pre": _z(5, 6), "activation": "gelu"}
    assert HOST in _refused(ops.linear_act_bwd, **good)
    assert HOST not in _refused(ops.linear_act_bwd, **{**good, **kw})


@pytest.mark.parametrize("what", [None, 3, [1.0], "x"])
def test_no_tensor(what):
    """Something else than a tensor is a TypeError, as for PyTorch's own operators."""
    x, w, s = _z(5, 8), _z(6, 8), _z(5, dtype=torch.float32)
    for call in (lambda: ops.layernorm_fwd(what), lambda: ops.layernorm_bwd(what, x, s, s), lambda: ops.linear_act(what, w), lambda: ops.linear_act_bwd(_z(5, 6), x, what)):
        with pytest.raises(TypeError):
            call()
    if what is not None:
        with pytest.raises(TypeError):
            ops.layernorm_fwd(x, bias=what)
    with pytest.raises(TypeError):
        ops.layernorm_fwd(x, eps="small")


# ---- the C entry points: refused before any CUDA call --------------------------------------------
# (made-up addresses: not where a device could read them)
P = 0x1000
no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="a device is present")


def _norm_fwd(**kw):
    a = {"x": P, "ldx": 64, "w": P, "b": P, "y": P, "ldy": 64, "mean": P, "rstd": P, "rows": 4, "C": 64, "dtype": 0, "pt": 0, "eps": 1e-5, **kw}
    return _lib.load().bxl_layernorm_fwd(*a.values(), None)


@no_device
@pytest.mark.parametrize("kw", [{"x": None}, {"y": None}, {"rows": 0}, {"rows": -1}, {"C": 0}, {"C": (1 << 30) + 1}, {"ldy": 63}, {"ldx": -1}, {"mean": None}, {"rstd": None},
                                {"dtype": 3}, {"dtype": 2}, {"pt": 1}, {"eps": -1.0}, {"eps": float("nan")}, {"x": P + 1}, {"w": P + 1}, {"mean": P + 2}])
def test_c_layernorm_fwd_refuses(kw):
    assert _norm_fwd(**kw) < 0 and b"bxl_layernorm_fwd" in _lib.load().bxl_last_error()


@no_device
@pytest.mark.parametrize("kw", [{"dy": None}, {"x": None}, {"mean": None}, {"rstd": None}, {"dx": None}, {"rows": 0}, {"C": -8}, {"lddx": 8}, {"lddy": -64}, {"pt": 1},
                                {"dtype": -1}, {"dw": P + 1}, {"dx": P + 1}, {"ws": None, "rows": 4000}, {"ws": P + 8, "rows": 4000}, {"ws_bytes": 16, "rows": 4000}])
def test_c_layernorm_bwd_refuses(kw):
    a = {"dy": P, "lddy": 64, "x": P, "ldx": 64, "mean": P, "rstd": P, "w": P, "dx": P, "lddx": 64, "dw": P, "db": P, "rows": 4, "C": 64, "dtype": 0, "pt": 0,
         "ws": P, "ws_bytes": 1 << 20, **kw}
    assert _lib.load().bxl_layernorm_bwd(*a.values(), None) < 0 and b"bxl_layernorm_bwd" in _lib.load().bxl_last_error()


def _linear(**kw):
    a = _lib.LinearArgs()
    base = {"x": P, "ldx": 64, "weight": P, "ldw": 64, "y": P, "ldy": 64, "dy": P, "lddy": 64, "dx": P, "lddx": 64, "dweight": P, "lddw": 64, "dbias": P,
            "M": 32, "N": 64, "K": 64, "dtype": 0, "act": 0, "workspace": P, "workspace_bytes": 1 << 20}
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return C.byref(a)


BOTH = [{"x": None}, {"weight": None}, {"M": 0}, {"N": -1}, {"K": 0}, {"M": (1 << 30) + 1}, {"dtype": 2}, {"dtype": 7}, {"act": 6}, {"act": -1}, {"x": P + 1}, {"bias": P + 1}, {"ldx": -1}]


@no_device
@pytest.mark.parametrize("kw", BOTH + [{"y": None}, {"ldy": 63}, {"pre": P, "ldp": 8}, {"ldx": 65, "workspace": None}, {"ldx": 65, "workspace_bytes": 64}])
def test_c_linear_act_fwd_refuses(kw):
    l = _lib.load()
    assert l.bxl_linear_act_fwd(_linear(**kw), None, None) < 0 and b"bxl_linear_act_fwd" in l.bxl_last_error()


@no_device
@pytest.mark.parametrize("kw", BOTH + [{"dy": None}, {"act": 3}, {"lddx": 63}, {"lddw": 0}, {"lddy": -1}, {"workspace": None, "M": 1000}, {"workspace": P + 4, "M": 1000}, {"workspace_bytes": 8, "M": 1000}])
def test_c_linear_act_bwd_refuses(kw):
    l = _lib.load()
    assert l.bxl_linear_act_bwd(_linear(**kw), None, None) < 0 and b"bxl_linear_act_bwd" in l.bxl_last_error()


@pytest.mark.parametrize("kw,nbytes", [({}, 0), ({"ldx": 68}, 32 * 64 * 2), ({"ldw": 65}, 64 * 64 * 2), ({"x": P + 2, "ldx": 0}, 32 * 64 * 2), ({"M": 8, "ldx": 65}, 0),
                                       ({"K": 63}, 0), ({"K": 63, "ldx": 63}, 32 * 64 * 2)])
def test_workspace_of_the_forward_pass(kw, nbytes):
    """Copies only of operands whose rows are not 16-byte aligned, and none for a few rows."""
    assert _lib.load().bxl_linear_act_fwd_workspace_bytes(_linear(**kw)) == nbytes


def test_workspace_leaves_room_to_align():
    """Partial sums are stored 32 bytes at a time: 16 bytes more than they take, for a 32-byte boundary in a workspace that is 16-byte aligned."""
    l = _lib.load()
    sliced = l.bxl_linear_act_fwd_workspace_bytes(_linear(M=60, N=24, K=3528, ldx=3528, ldw=3528, ldy=24))
    assert sliced > 60 * 32 * 4 * 2 and sliced % 32 == 16
    sums = l.bxl_layernorm_bwd_workspace_bytes(600, 8192)
    assert sums > 2 * 8192 * 4 and sums % 32 == 16 and l.bxl_layernorm_bwd_workspace_bytes(5, 8192) == 0


def test_out_that_requires_a_gradient_is_refused():
    """As PyTorch refuses it: what is written would be missing from the graph.  Without grad mode there is none."""
    for call in (lambda out: ops.layernorm_fwd(_z(5, 8), out=out), lambda out: ops.linear_act(_z(5, 4), _z(8, 4), out=out)):
        leaf = _z(5, 8).requires_grad_()
        assert "out requires a gradient" in _refused(call, out=leaf) and "out requires a gradient" in _refused(call, out=leaf * 2)
        with torch.no_grad():
            assert HOST in _refused(call, out=leaf)
        assert HOST in _refused(call, out=leaf.detach())


def test_workspace_of_the_backward_norm():
    """One row of sums for each of at most 148 blocks (the SMs of the device; the library counts 148 without one)."""
    l = _lib.load()
    sms = torch.cuda.get_device_properties(0).multi_processor_count if torch.cuda.is_available() else 148
    for rows in (513, 4096, 1 << 40):
        assert l.bxl_layernorm_bwd_workspace_bytes(rows, 640) == sms * 2 * 640 * 4 + 16
