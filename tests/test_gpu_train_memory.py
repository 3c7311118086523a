"""The training operators write to their results and their workspace, and to nothing beside them."""
import ctypes as C

import pytest
import torch

from tests._util import cuda_or_skip

pytestmark = pytest.mark.gpu
GUARD, FILL = 4 << 20, 0xA5


class _Arena:
    """Buffers with filled room in front of and behind each."""

    def __init__(self, sizes):
        self.at, end = {}, GUARD
        for name, n in sizes.items():
            self.at[name] = (end, n)
            end += (n + 255) // 256 * 256 + GUARD
        self.data = torch.full((end,), FILL, dtype=torch.uint8, device="cuda")

    def ptr(self, name):
        return self.data.data_ptr() + self.at[name][0]

    def check(self):
        end = 0
        for name, (begin, n) in [*self.at.items(), ("the end", (self.data.numel(), 0))]:
            assert bool((self.data[end:begin] == FILL).all()), f"written in front of {name}"
            end = begin + n


def _lib():
    from basedxl_b200 import _lib

    return _lib, _lib.lib()


# dbias in shares of many rows, copied operands, results of any alignment, K in slices, two products in a launch, few rows
LINEAR = [(16000, 256, 6720), (4000, 64, 2048), (257, 72, 4096), (300, 77, 1280), (5000, 42, 33), (159, 34, 5832), (60, 3528, 24), (40, 490, 2304), (10, 5120, 64),
          (8, 1000, 130), (3, 3907, 17), (1024, 648, 1288), (2050, 640, 321)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("m,k,n", LINEAR)
def test_linear_layers(m, k, n, dtype):
    cuda_or_skip()
    _l, lib = _lib()
    rn = lambda *s: torch.randn(*s, device="cuda").to(dtype)
    x, w, b, dy, res = rn(m, k), rn(n, k), rn(n), rn(m, n), rn(m, n)
    a = _l.LinearArgs()
    a.x, a.ldx, a.weight, a.ldw, a.bias = x.data_ptr(), k, w.data_ptr(), k, b.data_ptr()
    a.M, a.N, a.K, a.dtype, a.act = m, n, k, 0 if dtype == torch.float16 else 1, 2
    launches = C.c_int(0)
    stream = torch.cuda.current_stream().cuda_stream

    def run(entry, query, names, others):
        for key, (size, ld) in {**names, **{o: (0, v[1]) for o, v in others.items()}}.items():
            setattr(a, {"y": "ldy", "pre": "ldp", "residual": "ldr", "dx": "lddx", "dweight": "lddw", "dy": "lddy"}.get(key, "ldr"), ld)
        for key, (t, _) in others.items():
            setattr(a, key, t.data_ptr())
        first = _Arena({key: size for key, (size, _) in names.items()})
        for key in names:
            setattr(a, key, first.ptr(key))
        need = query(C.byref(a))
        arena = _Arena({**{key: size for key, (size, _) in names.items()}, "workspace": max(need, 1)})
        for key in names:
            setattr(a, key, arena.ptr(key))
        a.workspace, a.workspace_bytes = arena.ptr("workspace"), need
        _l.check(entry(C.byref(a), C.byref(launches), stream), lib)
        torch.cuda.synchronize()
        arena.check()
        return arena

    fwd = run(lib.bxl_linear_act_fwd, lib.bxl_linear_act_fwd_workspace_bytes, {"y": (2 * m * n, n), "pre": (2 * m * n, n)}, {"residual": (res, n)})
    begin, size = fwd.at["pre"]
    pre = fwd.data[begin : begin + size].clone()
    a.y = None
    run(lib.bxl_linear_act_bwd, lib.bxl_linear_act_bwd_workspace_bytes, {"dx": (2 * m * k, k), "dweight": (2 * n * k, k), "dbias": (2 * n, n)}, {"dy": (dy, n), "pre": (pre, n)})
    _l.device_status()


NORM = [(154, 2048), (513, 640), (20000, 64), (4001, 320), (1701, 643), (3000, 1280), (1025, 5120), (530, 13440), (600, 20000), (520, 70001), (40000, 33)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("rows,c", NORM)
def test_layernorm(rows, c, dtype):
    cuda_or_skip()
    _l, lib = _lib()
    rn = lambda *s: torch.randn(*s, device="cuda").to(dtype)
    x, w, b, dy = rn(rows, c), rn(c), rn(c), rn(rows, c)
    code, size = (1, 2) if dtype == torch.bfloat16 else (2, 4)
    stream = torch.cuda.current_stream().cuda_stream
    f = _Arena({"y": size * rows * c, "mean": 4 * rows, "rstd": 4 * rows})
    _l.check(lib.bxl_layernorm_fwd(x.data_ptr(), c, w.data_ptr(), b.data_ptr(), f.ptr("y"), c, f.ptr("mean"), f.ptr("rstd"), rows, c, code, code, 1e-5, stream), lib)
    need = lib.bxl_layernorm_bwd_workspace_bytes(rows, c)
    g = _Arena({"dx": size * rows * c, "dweight": size * c, "dbias": size * c, "workspace": max(need, 1)})
    _l.check(lib.bxl_layernorm_bwd(dy.data_ptr(), c, x.data_ptr(), c, f.ptr("mean"), f.ptr("rstd"), w.data_ptr(), g.ptr("dx"), c, g.ptr("dweight"), g.ptr("dbias"),
                                   rows, c, code, code, g.ptr("workspace") if need else None, need, stream), lib)
    torch.cuda.synchronize()
    f.check()
    g.check()
    _l.device_status()


def test_two_streams_at_once():
    """Calls of every operator on two streams beside one another give what they give one after the other."""
    cuda_or_skip()
    from basedxl_b200 import ops

    def inputs(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rn = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()
        return [(rn(m, k), rn(n, k) * k**-0.5, rn(n), rn(m, n), rn(k)) for m, k, n in ((700, 1280, 640), (2500, 48, 40), (5, 320, 1280), (300, 321, 643))]

    def step(sets):
        out = []
        for x, w, b, dy, gain in sets:
            h, mean, rstd = ops.layernorm_fwd(x, gain, None, want_stats=True)
            y, pre = ops.linear_act(h, w, b, activation="gelu", residual=dy, want_pre=True)
            dh, dw, db = ops.linear_act_bwd(dy, h, w, pre, activation="gelu")
            out += [y, dw, db, *ops.layernorm_bwd(dh, x, mean, rstd, gain)]
        return out

    sets = [inputs(1), inputs(2)]
    want = [step(s) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(step(sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for once in got[i]:
            assert all(torch.equal(p, q) for p, q in zip(once, want[i]))


class _Shifted(_Arena):
    """The workspace lies 16 bytes behind a 32-byte boundary."""

    def __init__(self, sizes):
        super().__init__({name: n + 16 if name == "workspace" else n for name, n in sizes.items()})
        if "workspace" in self.at:
            self.at["workspace"] = (self.at["workspace"][0] + 16, sizes["workspace"])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("m,k,n", LINEAR)
def test_linear_layers_any_workspace(m, k, n, dtype, monkeypatch):
    """16-byte alignment is all that the workspace needs."""
    monkeypatch.setitem(globals(), "_Arena", _Shifted)
    test_linear_layers(m, k, n, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("rows,c", NORM + [(530, 8192), (530, 12288), (530, 6152)])
def test_layernorm_any_workspace(rows, c, dtype, monkeypatch):
    monkeypatch.setitem(globals(), "_Arena", _Shifted)
    test_layernorm(rows, c, dtype)
