"""LayerNorm forward and backward through the public entry points, against plain forms in 64 bits."""
import pytest
import torch

from tests import _plain
from tests._util import cuda_or_skip

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]
EPS = 1e-5


def _ops():
    from basedxl_b200 import _lib, ops

    return _lib, ops


def _inputs(rows, c, dtype, param_dtype=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=g)
    x = (rn(rows, c) * rn(c).mul(0.5).exp() + rn(rows, 1)).to(dtype)
    pt = param_dtype or dtype
    return x, (rn(c) * 0.2 + 1).to(pt), (rn(c) * 0.2).to(pt), rn(rows, c).to(dtype)


def _check(x, w, b, dy, want_dbias=True):
    _lib, ops = _ops()
    y, by, mean, bm, rstd, br = _plain.norm(x, w, b, EPS)
    got = ops.layernorm_fwd(x, w, b, EPS, want_stats=True)
    for v, want, bound, what in zip(got, (y, mean, rstd), (by, bm, br), ("y", "mean", "rstd")):
        _plain.within(v, want, bound, what)
    assert torch.equal(ops.layernorm_fwd(x, w, b, EPS), got[0])
    dx, dw, db = ops.layernorm_bwd(dy, x, got[1], got[2], w, want_dbias=want_dbias)
    want = _plain.norm_grad(dy, x, got[1], got[2], w)
    _plain.within(dx.flatten(0, -2), want[0], want[1], "dx")
    if w is not None:
        _plain.within(dw, want[2], want[3], "dweight")
    else:
        assert dw is None
    if want_dbias:
        _plain.within(db, want[4], want[5], "dbias")
    else:
        assert db is None
    _lib.device_status()


SHAPES = [(1, 1), (3, 2), (5, 7), (9, 8), (77, 31), (64, 64), (1, 255), (9, 256), (10, 257), (1, 320), (300, 320), (257, 640), (9, 648), (154, 768),
          (1, 1280), (77, 1280), (130, 1285), (2, 2048), (33, 2049), (3, 4096), (600, 4104), (2, 5120), (3, 8192), (2, 8199), (3, 10240), (2, 16384),
          (2, 16387), (3, 20008), (2, 40000), (2, 70001), (5000, 64), (3000, 40), (2500, 1280), (20011, 33)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,c", SHAPES)
def test_against_64_bits(rows, c, dtype):
    cuda_or_skip()
    _check(*_inputs(rows, c, dtype))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows,c", [(5, 7), (77, 640), (154, 2048), (9, 1285)])
def test_fp32_weights(rows, c, dtype):
    cuda_or_skip()
    _check(*_inputs(rows, c, dtype, torch.float32))


MANY = [(8009, 136), (4001, 320), (2101, 512), (1701, 648), (1501, 768), (1201, 1152), (1101, 1280), (801, 1608), (601, 2048), (601, 2560), (601, 4096),
        (600, 5120), (530, 8192), (520, 12000), (517, 16000), (513, 20000), (1701, 643), (601, 2049), (530, 8190)]


@pytest.mark.parametrize("dtype,param", [(torch.float16, torch.float16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)], ids=str)
@pytest.mark.parametrize("rows,c", MANY)
def test_many_rows(rows, c, dtype, param):
    """Every width of a team and number of vectors of a thread, with a last unit that is not full."""
    cuda_or_skip()
    _check(*_inputs(rows, c, dtype, param))


@pytest.mark.parametrize("rows,c", [(4001, 320), (2101, 512), (801, 1608), (601, 4096), (1701, 643)])
def test_many_rows_apart(rows, c):
    """Rows of a wider tensor, between values that are not to be read.  Rows of whole 16-byte vectors give the same bits as a copy of them;
    others are summed in another order where they do not lie back to back, and are held to the bounds that cover any order."""
    cuda_or_skip()
    _, ops = _ops()
    x, w, b, dy = _inputs(rows, c, torch.bfloat16)
    wide = torch.full((rows, 2 * c + 8), float("nan"), device="cuda", dtype=x.dtype)
    apart = wide[:, 8 : 8 + c]
    apart.copy_(x)
    _check(apart, w, b, dy)
    if c % 8 == 0:
        want = ops.layernorm_fwd(x, w, b, EPS, want_stats=True)
        got = ops.layernorm_fwd(apart, w, b, EPS, want_stats=True)
        want += ops.layernorm_bwd(dy, x, *want[1:], w)
        got += ops.layernorm_bwd(dy, apart, *got[1:], w)
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("dtype,param", [(torch.float16, torch.float16), (torch.bfloat16, torch.float32)], ids=str)
@pytest.mark.parametrize("rows,c", [(240007, 64), (470003, 40), (115003, 128), (60011, 512), (60013, 640), (30011, 1024)])
def test_units_of_several_rows(rows, c, dtype, param):
    """Rows enough for several of them to share a stage of the ring, the last one not full; and rows of a wider tensor."""
    cuda_or_skip()
    x, w, b, dy = _inputs(rows, c, dtype, param)
    _check(x, w, b, dy)
    _check(torch.cat([x, x], dim=1)[:, c:], w, b, dy)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,c", [(19003, 643), (19001, 601), (38003, 301), (76003, 131), (9601, 1285), (5003, 1819), (600, 12001), (2401, 9001)])
def test_many_rows_of_any_length(rows, c, dtype):
    cuda_or_skip()
    _check(*_inputs(rows, c, dtype))


@pytest.mark.parametrize("rows,c", [(40, 1285), (4001, 320), (801, 1608), (1701, 643), (60011, 640)])
def test_repeated_rows(rows, c):
    cuda_or_skip()
    x, w, b, dy = _inputs(rows, c, torch.float16)
    _check(x[:1].expand_as(x), w, b, dy)
    _check(x, w, b, dy[:1].expand_as(dy))


@pytest.mark.parametrize("rows,c", [(40, 1285), (4001, 320), (801, 1608), (601, 4096), (1701, 643), (513, 20000)])
def test_in_place(rows, c):
    cuda_or_skip()
    _, ops = _ops()
    x, w, b, _ = _inputs(rows, c, torch.float16, torch.float32)
    want = ops.layernorm_fwd(x, w, b, EPS)
    assert ops.layernorm_fwd(x, w, b, EPS, out=x) is not want and torch.equal(x, want)


@pytest.mark.parametrize("c", [5, 640, 2048, 17000])
def test_absent_weight_or_bias(c):
    cuda_or_skip()
    _lib, ops = _ops()
    x, w, b, dy = _inputs(7, c, torch.float16)
    _check(x, None, None, dy)
    _check(x, w, None, dy, want_dbias=False)
    _check(x, None, b, dy)
    stats = ops.layernorm_fwd(x, w, b, EPS, want_stats=True)[1:]
    full = ops.layernorm_bwd(dy, x, *stats, w)
    dx, dw, db = ops.layernorm_bwd(dy, x, *stats, w, want_dweight=False)
    assert dw is None and torch.equal(dx, full[0]) and torch.equal(db, full[2])
    dx, dw, db = ops.layernorm_bwd(dy, x, *stats, w, want_dweight=False, want_dbias=False)
    assert dw is None and db is None and torch.equal(dx, full[0])


@pytest.mark.parametrize("layout", ["slice", "odd slice", "one row", "columns first", "every second column", "three axes", "one axis"])
@pytest.mark.parametrize("c", [64, 640, 2056])
def test_layouts(layout, c):
    cuda_or_skip()
    x, w, b, dy = _inputs(24, c, torch.bfloat16)
    wide = torch.zeros(24, 2 * c + 16, device="cuda", dtype=x.dtype)
    if layout == "slice":
        wide[:, 8 : 8 + c] = x
        x = wide[:, 8 : 8 + c]
    elif layout == "odd slice":
        wide[:, 3 : 3 + c] = x
        x = wide[:, 3 : 3 + c]
        dy = torch.cat([dy[:, :1], dy], dim=1)[:, 1:]
    elif layout == "one row":
        x, dy = x[:1].expand(24, c), dy[:1].expand(24, c)
    elif layout == "columns first":
        x = x.t().contiguous().t()
    elif layout == "every second column":
        wide[:, : 2 * c : 2] = x
        x = wide[:, : 2 * c : 2]
    elif layout == "three axes":
        x, dy = x.view(2, 12, c).transpose(0, 1), dy.view(2, 12, c).transpose(0, 1)
    else:
        x, dy = x[0], dy[0]
        y = _ops()[1].layernorm_fwd(x, w, b, EPS)
        assert y.shape == (c,)
        _check(x[None], w, b, dy[None])
        return
    _check(x, w, b, dy)


def test_empty():
    cuda_or_skip()
    _, ops = _ops()
    x = torch.empty(3, 0, 64, device="cuda", dtype=torch.float16)
    w = torch.ones(64, device="cuda", dtype=torch.float16)
    y, mean, rstd = ops.layernorm_fwd(x, w, w, want_stats=True)
    assert y.shape == x.shape and mean.shape == rstd.shape == (3, 0)
    dx, dw, db = ops.layernorm_bwd(x, x, mean, rstd, w)
    assert dx.shape == x.shape and not dw.any() and not db.any()


@pytest.mark.parametrize("c", [40, 1280, 1285, 5120, 20001])
def test_constant_rows_and_large_means(c):
    """No variance: the result is the bias.  A mean of 4096 steps above the values' spread costs no more than the plain sums may."""
    cuda_or_skip()
    _, ops = _ops()
    x, w, b, dy = _inputs(4, c, torch.float32)
    x[0], x[1] = 3.0, 0.0
    y = ops.layernorm_fwd(x, w, b, EPS)
    assert torch.equal(y[0], b) and torch.equal(y[1], b)
    x[2:] += 4096
    _check(x[2:], w, b, dy[2:])


@pytest.mark.parametrize("c", [40, 1280, 1285, 5120])
def test_a_bad_row_stays_alone(c):
    cuda_or_skip()
    _, ops = _ops()
    x, w, b, dy = _inputs(20, c, torch.float16)
    clean = ops.layernorm_fwd(x, w, b, EPS, want_stats=True)
    gx = ops.layernorm_bwd(dy, x, *clean[1:], w)[0]
    bad = x.clone()
    bad[3, c // 2], bad[11, 0] = float("nan"), float("inf")
    got = ops.layernorm_fwd(bad, w, b, EPS, want_stats=True)
    rest = [i for i in range(20) if i not in (3, 11)]
    assert got[0][3].isnan().all() and got[0][11].isnan().any()
    for v, want in zip(got, clean):
        assert torch.equal(v[rest], want[rest])
    dx, dw, _ = ops.layernorm_bwd(dy, bad, *got[1:], w)
    assert torch.equal(dx[rest], gx[rest]) and dx[3].isnan().all() and dw.isnan().any()


def test_in_place_and_neighbours():
    """``out`` may be ``x``; nothing behind the last row is written."""
    cuda_or_skip()
    _, ops = _ops()
    for c in (40, 1280, 1285, 2056, 20008):
        x, w, b, _ = _inputs(13, c, torch.float16)
        want = ops.layernorm_fwd(x, w, b, EPS)
        room = torch.full((15, c), 7.0, device="cuda", dtype=torch.float16)
        ops.layernorm_fwd(x, w, b, EPS, out=room[1:14])
        assert torch.equal(room[1:14], want) and (room[0] == 7).all() and (room[14] == 7).all()
        assert ops.layernorm_fwd(x, w, b, EPS, out=x) is x and torch.equal(x, want)


def test_rows_past_32_bit_offsets():
    cuda_or_skip()
    _, ops = _ops()
    room = torch.empty(2_400_000_000, device="cuda", dtype=torch.float16)
    x, w, b, dy = _inputs(3, 640, torch.float16)
    far = room.as_strided((3, 640), (1_150_000_000, 1))
    far.copy_(x)
    y, mean, rstd = ops.layernorm_fwd(far, w, b, EPS, want_stats=True)
    assert torch.equal(y, ops.layernorm_fwd(x, w, b, EPS))
    assert all(torch.equal(p, q) for p, q in zip(ops.layernorm_bwd(dy, far, mean, rstd, w), ops.layernorm_bwd(dy, x, mean, rstd, w)))


@pytest.mark.parametrize("rows,c", [(40, 640), (33, 1285), (9, 17000)])
def test_same_bits_every_time_and_from_graphs(rows, c):
    """Two captured graphs, replayed in turn on a stream of their own with new inputs, give what eager calls give."""
    cuda_or_skip()
    _, ops = _ops()
    sets = [_inputs(rows, c, torch.bfloat16, torch.float32, seed=s) for s in (1, 2, 3)]

    def step(x, w, b, dy):
        y, mean, rstd = ops.layernorm_fwd(x, w, b, EPS, want_stats=True)
        return (y, mean, rstd, *ops.layernorm_bwd(dy, x, mean, rstd, w))

    want = [step(*s) for s in sets]
    assert all(torch.equal(p, q) for s, v in zip(sets, want) for p, q in zip(step(*s), v))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for s in sets[:2]:
            held = [t.clone() for t in s]
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                got = step(*held)
            graphs.append((g, held, got))
        for k in (2, 0, 1):
            for g, held, got in graphs:
                for t, v in zip(held, sets[k]):
                    t.copy_(v)
                g.replay()
            for _, _, got in graphs:
                side.synchronize()
                assert all(torch.equal(p, q) for p, q in zip(got, want[k]))


@pytest.mark.parametrize("rows,c", [(6, 40), (5, 1285), (3, 5120)])
def test_gradients_against_differences(rows, c):
    """<gradient, v> of sum(y dy) against a central difference of the fp32 forward kernel along v, summed in 64 bits.  The
    difference's own error: 8 U |y| from each rounded result, and the h^2 term, taken from the same difference in 64 bits."""
    cuda_or_skip()
    _, ops = _ops()
    x, w, b, dy = _inputs(rows, c, torch.float32)
    _, mean, rstd = ops.layernorm_fwd(x, w, b, EPS, want_stats=True)
    grads = ops.layernorm_bwd(dy, x, mean, rstd, w)
    g = torch.Generator(device="cuda").manual_seed(5)
    for i, grad in enumerate(grads):
        v = torch.randn(grad.shape, device="cuda", generator=g)
        h = 2.0**-6
        args = [[t.clone() for t in (x, w, b)] for _ in range(2)]
        args[0][i] += h * v
        args[1][i] -= h * v
        step = (args[0][i].double() - args[1][i].double())       # as rounded
        f = [(ops.layernorm_fwd(*a, EPS).double() * dy.double()).sum() for a in args]
        plain = [_plain.norm(*a, EPS) for a in args]
        f64 = [(p[0] * dy.double()).sum() for p in plain]
        slope64 = (_plain_grad(x, w, b, dy)[i] * step).sum()
        got = (grad.double() * step).sum()
        bound = (f64[0] - f64[1] - slope64).abs() + sum(((p[1] + U_HALF * p[0].abs()) * dy.double().abs()).sum() for p in plain)
        own = _plain.norm_grad(dy, x, mean, rstd, w)[2 * i + 1] if i else _plain.norm_grad(dy, x, mean, rstd, w)[1].view_as(grad)
        bound = bound + ((own + 4 * U_HALF * grad.double().abs()) * step.abs()).sum()
        assert (got - (f[0] - f[1])).abs() <= bound


U_HALF = 2.0**-24


def _plain_grad(x, w, b, dy):
    leaves = [t.double().requires_grad_() for t in (x, w, b)]
    y = torch.nn.functional.layer_norm(leaves[0], w.shape, leaves[1], leaves[2], EPS)
    return torch.autograd.grad(y, leaves, dy.double())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("rows,c", [(20, 320), (4001, 320), (801, 1608), (1701, 643), (60011, 640), (513, 20000)])
def test_mean_of_infinite_rows(rows, c, dtype):
    """The mean of a row is infinite where its sum is, for few rows and for many; its other results are NaN, other rows as they were."""
    cuda_or_skip()
    _lib, ops = _ops()
    x, w, b, _ = _inputs(rows, c, dtype)
    clean = ops.layernorm_fwd(x, w, b, EPS, want_stats=True)
    x = x.clone()
    inf = float("inf")
    x[3, 5], x[7, 0], x[rows - 1, c - 1], x[9, 1], x[9, 2] = inf, -inf, inf, inf, -inf
    y, mean, rstd = ops.layernorm_fwd(x, w, b, EPS, want_stats=True)
    assert mean[3] == inf and mean[7] == -inf and mean[rows - 1] == inf and mean[9].isnan()
    hit = [3, 7, 9, rows - 1]
    assert y[hit].isnan().all() and rstd[hit].isnan().all()
    rest = torch.ones(rows, dtype=torch.bool, device="cuda")
    rest[hit] = False
    assert all(torch.equal(p[rest], q[rest]) for p, q in zip((y, mean, rstd), clean))
    _lib.device_status()


@pytest.mark.parametrize("rows,c,apart,kernels", [(5, 97, True, 1), (600, 97, True, 3), (600, 96, False, 2), (600, 20000, False, 3), (513, 11600, False, 3)])
def test_counted_launches(rows, c, apart, kernels):
    """One kernel for few rows, two with the column sums, three where the rows have no ring; one without column sums."""
    cuda_or_skip()
    _lib, ops = _ops()
    x = torch.randn(rows, c + 3, device="cuda")[:, 1 : c + 1]
    x = x if apart else x.contiguous()
    w = torch.ones(c, device="cuda")
    _, mean, rstd = ops.layernorm_fwd(x, w, want_stats=True)
    for want, n in (({}, kernels), ({"want_dbias": False}, kernels), ({"want_dweight": False, "want_dbias": False}, 1)):
        before = _lib.launches
        ops.layernorm_bwd(x, x, mean, rstd, w, **want)
        assert _lib.launches - before == n


@pytest.mark.parametrize("rows,c", [(30011, 1280), (30011, 1408), (30011, 1792)])
def test_many_rows_of_five_to_seven_vectors(rows, c):
    """Enough rows for units of several, at the widths up to which a warp's threads hold a row."""
    cuda_or_skip()
    _check(*_inputs(rows, c, torch.float16))
