"""Linear layers with an activation, forward and backward, through the public entry points, against plain forms in 64 bits."""
import pytest
import torch

from tests import _plain
from tests._util import cuda_or_skip

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh", "quick_gelu"]


def _ops():
    from basedxl_b200 import _lib, ops

    return _lib, ops


def _inputs(m, k, n, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s, scale=1.0: (torch.randn(*s, device="cuda", generator=g) * scale).to(dtype)
    return {"x": rn(m, k), "weight": rn(n, k, scale=k**-0.5), "bias": rn(n, scale=0.3), "residual": rn(m, n), "dy": rn(m, n)}


def _check_fwd(s, act, bias=True, residual=True):
    _, ops = _ops()
    b, r = s["bias"] if bias else None, s["residual"] if residual else None
    want = _plain.linear(s["x"], s["weight"], b, act, r)
    y, pre = ops.linear_act(s["x"], s["weight"], b, activation=act, residual=r, want_pre=True)
    _plain.within(y, want[0], want[1], "y")
    _plain.within(pre, want[2], want[3], "pre")
    assert torch.equal(ops.linear_act(s["x"], s["weight"], b, activation=act, residual=r), y)
    return pre


def _check_bwd(s, act, pre):
    _, ops = _ops()
    got = ops.linear_act_bwd(s["dy"], s["x"], s["weight"], pre, activation=act)
    want = _plain.linear_grad(s["dy"], s["x"], s["weight"], pre, act)
    for i, what in enumerate(("dx", "dweight", "dbias")):
        _plain.within(got[i].view(want[2 * i].shape), want[2 * i], want[2 * i + 1], what)
    return got


SHAPES = [(1, 1, 1), (1, 320, 1280), (2, 320, 1280), (2, 1280, 640), (3, 7, 5), (4, 256, 33), (5, 1000, 130), (6, 65, 64), (7, 2048, 9), (8, 640, 1283), (9, 64, 64),
          (16, 8, 32), (33, 1, 7), (77, 2048, 1280), (128, 64, 256), (129, 65, 33), (200, 104, 1000), (257, 1003, 1501), (300, 1280, 640), (1024, 320, 1288),
          (2050, 640, 328), (5000, 17, 19), (40, 5120, 8), (13000, 42, 33), (159, 34, 5832), (60, 3528, 24), (300, 4999, 40), (6000, 744, 16)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_against_64_bits(m, k, n, dtype):
    cuda_or_skip()
    _lib, _ = _ops()
    s = _inputs(m, k, n, dtype)
    act = ACTS[(m + k + n) % len(ACTS)]
    pre = _check_fwd(s, act)
    _check_bwd(s, act, pre)
    _lib.device_status()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,k,n", [(2, 320, 72), (130, 128, 200), (150, 77, 99)])
def test_activations(m, k, n, act, dtype):
    cuda_or_skip()
    s = _inputs(m, k, n, dtype)
    s["weight"] = s["weight"] * 3  # pre-activations out to +-10, where the tails are
    for bias, residual in ((True, False), (False, True), (False, False)):
        pre = _check_fwd(s, act, bias, residual)
    _check_bwd(s, act, pre)


@pytest.mark.parametrize("tiles", [(32, 1, 0), (64, 1, 0), (128, 1, 0), (256, 1, 0), (64, 2, 0), (128, 4, 0), (256, 2, 0), (128, 1, 1), (256, 1, 1)], ids=str)
@pytest.mark.parametrize("m,k,n", [(300, 448, 520), (300, 449, 519)])
def test_every_tiling(m, k, n, tiles):
    cuda_or_skip()
    _lib, _ = _ops()
    l = _lib.lib()
    s = _inputs(m, k, n, torch.bfloat16)
    try:
        _lib.check(l.bxl_debug_force_tiles(*tiles), l, kernels=0)
        _check_bwd(s, "gelu", _check_fwd(s, "gelu"))
    finally:
        l.bxl_debug_force_tiles(0, 0, -1)
    _lib.device_status()


@pytest.mark.parametrize("tiles", [(32, 1, 0), (96, 1, 0), (160, 1, 0), (224, 1, 0), (96, 1, 1), (192, 1, 1), (224, 1, 1), (192, 2, 0), (0, 0, -1)], ids=str)
@pytest.mark.parametrize("m,k,n", [(300, 456, 520), (8000, 96, 648)])
def test_any_width(m, k, n, tiles):
    """Tiles that are no multiple of the 64 columns that an operand is fetched in, one and many of them for each CTA."""
    cuda_or_skip()
    _lib, _ = _ops()
    l = _lib.lib()
    s = _inputs(m, k, n, torch.bfloat16)
    _lib.check(l.bxl_debug_force_tiles(*tiles), l, kernels=0)
    try:
        pre = _check_fwd(s, "silu")
        _check_bwd(s, "silu", pre)
        _lib.device_status()
    finally:
        _lib.check(l.bxl_debug_force_tiles(0, 0, -1), l, kernels=0)


@pytest.mark.parametrize("m", [3, 140])
@pytest.mark.parametrize("layout", ["slice", "odd slice", "one row", "columns first", "three axes", "one axis"])
def test_layouts(layout, m):
    cuda_or_skip()
    _, ops = _ops()
    k, n = 136, 200
    s = _inputs(m, k, n, torch.float16)

    def moved(t, at):
        room = torch.zeros(t.shape[0], t.shape[1] + 16, device="cuda", dtype=t.dtype)
        room[:, at : at + t.shape[1]] = t
        return room[:, at : at + t.shape[1]]

    if layout in ("slice", "odd slice"):
        s = {q: moved(t, 8 if layout == "slice" else 3) if t.dim() == 2 else torch.cat([t[:1], t])[1:] for q, t in s.items()}
    elif layout == "one row":
        s = {q: t[:1].expand_as(t) if t.dim() == 2 else t for q, t in s.items()}
    elif layout == "columns first":
        s = {q: t.t().contiguous().t() if t.dim() == 2 else t for q, t in s.items()}
    elif layout == "three axes":
        flat = dict(s)
        s = {q: torch.stack([t, t.flip(0)]).transpose(0, 1) if q in ("x", "residual", "dy") else t for q, t in s.items()}
        flat = {q: s[q].reshape(-1, s[q].shape[-1]) if s[q].dim() == 3 else s[q] for q in s}
        y, pre = ops.linear_act(s["x"], s["weight"], s["bias"], activation="silu", residual=s["residual"], want_pre=True)
        assert y.shape == pre.shape == (m, 2, n)
        assert torch.equal(y.view(-1, n), ops.linear_act(flat["x"], s["weight"], s["bias"], activation="silu", residual=flat["residual"]))
        got, want = ops.linear_act_bwd(s["dy"], s["x"], s["weight"], pre, "silu"), ops.linear_act_bwd(flat["dy"], flat["x"], s["weight"], pre.view(-1, n), "silu")
        assert got[0].shape == (m, 2, k) and all(torch.equal(p.view(q.shape), q) for p, q in zip(got, want))
        return
    elif layout == "one axis":
        y, pre = ops.linear_act(s["x"][0], s["weight"], s["bias"], activation="silu", want_pre=True)
        assert y.shape == pre.shape == (n,)
        one = {q: t[:1] if q in ("x", "residual", "dy") else t for q, t in s.items()}
        got = ops.linear_act_bwd(s["dy"][0], s["x"][0], s["weight"], pre, "silu")
        assert all(torch.equal(p.view(q.shape), q) for p, q in zip(got, _check_bwd(one, "silu", pre[None])))
        return
    pre = _check_fwd(s, "silu")
    _check_bwd(s, "silu", moved(pre, 5) if layout == "odd slice" else pre)
    _check_bwd(s, "none", None)


@pytest.mark.parametrize("m,k,n", [(3, 320, 640), (140, 320, 640), (140, 72, 99), (20, 2048, 64), (3000, 64, 264)])
def test_repeated_rows(m, k, n):
    """Broadcast rows, one memory for all of them, in the place of every input that has rows."""
    cuda_or_skip()
    _lib, ops = _ops()
    s = _inputs(m, k, n, torch.bfloat16)
    one = {name: s[name][:1].expand_as(s[name]) for name in ("x", "residual", "dy")}
    pre = _check_fwd({**s, "residual": one["residual"]}, "silu")
    _check_fwd({**s, "x": one["x"]}, "gelu")
    _check_bwd({**s, "dy": one["dy"]}, "silu", pre)
    _check_bwd({**s, "x": one["x"], "dy": one["dy"]}, "none", None)
    _check_bwd(s, "relu", pre[:1].expand_as(pre))
    _lib.device_status()


@pytest.mark.parametrize("m,k,n", [(68, 2240, 64), (16, 2752, 832), (820, 5032, 88), (517, 2759, 16), (11, 2189, 184), (4096, 320, 2560), (300, 640, 640), (5, 320, 64)])
def test_same_bits_with_and_without(m, k, n):
    """Neither keeping the value before the activation nor a residual of zeros changes the result."""
    cuda_or_skip()
    _, ops = _ops()
    s = _inputs(m, k, n, torch.bfloat16)
    y = ops.linear_act(s["x"], s["weight"], s["bias"], activation="silu")
    zeros = torch.zeros_like(y)
    assert torch.equal(ops.linear_act(s["x"], s["weight"], s["bias"], activation="silu", want_pre=True)[0], y)
    assert torch.equal(ops.linear_act(s["x"], s["weight"], s["bias"], activation="silu", residual=zeros), y)
    assert torch.equal(ops.linear_act(s["x"], s["weight"], s["bias"], activation="silu", residual=zeros, want_pre=True)[0], y)


def test_empty_and_wanted():
    cuda_or_skip()
    _, ops = _ops()
    s = _inputs(20, 64, 96, torch.float16)
    none = {q: t[:0] if q in ("x", "dy", "residual") else t for q, t in s.items()}
    y, pre = ops.linear_act(none["x"], s["weight"], s["bias"], activation="gelu", residual=none["residual"], want_pre=True)
    assert y.shape == pre.shape == (0, 96)
    dx, dw, db = ops.linear_act_bwd(none["dy"], none["x"], s["weight"], pre, "gelu")
    assert dx.shape == (0, 64) and not dw.any() and not db.any()
    for act in ("none", "gelu"):
        pre = ops.linear_act(s["x"], s["weight"], s["bias"], activation=act, want_pre=True)[1]
        full = ops.linear_act_bwd(s["dy"], s["x"], s["weight"], pre, act)
        for want in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 0, 0)):
            got = ops.linear_act_bwd(s["dy"], s["x"], s["weight"], pre, act, *map(bool, want))
            assert all((g is None) if not q else torch.equal(g, f) for g, f, q in zip(got, full, want))


@pytest.mark.parametrize("m", [2, 64])
@pytest.mark.parametrize("act", ACTS)
def test_infinite_and_missing_values(act, m):
    """Infinite pre-activations give the limits (to 2^-50: a sigmoid is not formed below 2^-60), NaN stays in its row and column."""
    cuda_or_skip()
    _, ops = _ops()
    s = _inputs(m, 64, 40, torch.bfloat16)
    x = s["x"].clone()
    x[0], x[1] = 0, 0
    x[0, 0], x[1, 1] = float("inf"), float("nan")
    w = s["weight"].clone()
    w[:, 1:] = s["weight"][:, 1:].abs() + 0.125
    w[:, 0] = 1.0
    w[20:, 0] = -1.0
    x[0, 1:] = 0
    y, pre = ops.linear_act(x, w, None, activation=act, want_pre=True)
    assert (pre[0, :20] == float("inf")).all() and (pre[0, 20:] == float("-inf")).all() and pre[1].isnan().all() and y[1].isnan().all()
    assert (y[0, :20] == float("inf")).all()
    assert (y[0, 20:] == float("-inf")).all() if act == "none" else (y[0, 20:].abs() < 2.0**-50).all()
    dy = torch.ones_like(y)
    _, _, db = ops.linear_act_bwd(dy[:1], x[:1], w, pre[:1], act)
    assert (db[:20] == 1).all() and ((db[20:] - (1 if act == "none" else 0)).abs() < 2.0**-50).all()
    if m > 2:
        assert torch.equal(y[2:], ops.linear_act(s["x"], w, None, activation=act)[2:])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,k,n", [(2, 64, 48), (64, 64, 48), (300, 64, 48), (300, 64, 45), (60, 3528, 24), (1000, 64, 512)])
def test_a_missing_value_stays_in_its_column(m, k, n, act, dtype):
    """A NaN in one element of the bias, in a row of the weight or in one element of ``pre``: every other column of the results, and
    every other row of ``dweight``, is what it is without."""
    cuda_or_skip()
    _lib, ops = _ops()
    s = _inputs(m, k, n, dtype)
    nan, lost = float("nan"), [3, 10, 17]
    rest = [j for j in range(n) if j not in lost]
    w, b = s["weight"].clone(), s["bias"].clone()
    b[3] = b[10] = nan
    w[17, k // 2] = nan
    want = _plain.linear(s["x"], s["weight"], s["bias"], act, None)
    y, pre = ops.linear_act(s["x"], w, b, activation=act, want_pre=True)
    assert y[:, lost].isnan().all() and pre[:, lost].isnan().all()
    _plain.within(y[:, rest], want[0][:, rest], want[1][:, rest], "y")
    _plain.within(pre[:, rest], want[2][:, rest], want[3][:, rest], "pre")
    if act == "none":   # its backward pass takes no pre
        return
    pre = ops.linear_act(s["x"], s["weight"], s["bias"], activation=act, want_pre=True)[1]
    want = _plain.linear_grad(s["dy"], s["x"], s["weight"], pre, act)
    bad = pre.clone()
    bad[0, 3] = bad[m - 1, 10] = bad[0, 17] = nan
    dx, dw, db = ops.linear_act_bwd(s["dy"], s["x"], s["weight"], bad, act)
    assert dx[[0, m - 1]].isnan().all() and dw[lost].isnan().all() and db[lost].isnan().all()
    if m > 2:
        _plain.within(dx[1 : m - 1], want[0][1 : m - 1], want[1][1 : m - 1], "dx")
    _plain.within(dw[rest], want[2][rest], want[3][rest], "dweight")
    _plain.within(db[rest], want[4][rest], want[5][rest], "dbias")
    _lib.device_status()


@pytest.mark.parametrize("m,k,n", [(4, 1003, 2400), (8, 640, 2400), (8, 65, 1280), (40, 1003, 640), (40, 640, 640)])
def test_inputs_of_the_kernel_before(m, k, n):
    """Rows and bias that the calls right before have written, over values that an earlier call of the same layer has read."""
    cuda_or_skip()
    _, ops = _ops()
    w, wb = _inputs(m, k, n, torch.float16)["weight"], _inputs(1, k, n, torch.float16, 7)["weight"]
    xs = [_inputs(m, k, n, torch.float16, seed)["x"] for seed in range(20)]
    want = []
    for x in xs:
        y = ops.layernorm_fwd(x)
        b = ops.linear_act(x[0], wb)
        torch.cuda.synchronize()
        want.append(ops.linear_act(y, w, b, activation="silu"))
        torch.cuda.synchronize()
    x, b, got = torch.empty_like(xs[0]), torch.empty(n, device="cuda", dtype=torch.float16), []
    for _ in range(5):
        for v in xs:
            x.copy_(v)
            ops.linear_act(x, w, b, activation="silu")
            ops.linear_act(x[0], wb, out=b)
            ops.layernorm_fwd(x, out=x)
            got.append(ops.linear_act(x, w, b, activation="silu"))
    assert all(torch.equal(p, q) for p, q in zip(got, want * 5))


def test_out_and_neighbours():
    """``out`` may be the residual; nothing behind the last row is written."""
    cuda_or_skip()
    _, ops = _ops()
    for m, k, n in ((2, 64, 48), (5, 33, 31), (140, 64, 200), (140, 64, 199)):
        s = _inputs(m, k, n, torch.float16)
        want = ops.linear_act(s["x"], s["weight"], s["bias"], activation="silu", residual=s["residual"])
        room = torch.full((m + 2, n), 7.0, device="cuda", dtype=torch.float16)
        ops.linear_act(s["x"], s["weight"], s["bias"], activation="silu", residual=s["residual"], out=room[1 : m + 1])
        assert torch.equal(room[1 : m + 1], want) and (room[0] == 7).all() and (room[m + 1] == 7).all()
        r = s["residual"].clone()
        assert ops.linear_act(s["x"], s["weight"], s["bias"], activation="silu", residual=r, out=r) is r and torch.equal(r, want)


def test_results_past_32_bit_offsets():
    cuda_or_skip()
    _lib, ops = _ops()
    m, k, n = 70_000, 16, 32_000
    s = {q: t for q, t in _inputs(1, k, n, torch.float16).items()}
    x = torch.randn(m, k, device="cuda").half()
    y, pre = ops.linear_act(x, s["weight"], s["bias"], activation="relu", want_pre=True)
    rows = [0, 1, 33_554, 67_107, 67_108, 67_109, m - 1]
    want = _plain.linear(x[rows], s["weight"], s["bias"], "relu", None)
    _plain.within(y[rows], want[0], want[1], "y")
    _plain.within(pre[rows], want[2], want[3], "pre")
    dx = ops.linear_act_bwd(y, x, s["weight"], pre, "relu", want_dweight=False, want_dbias=False)[0]
    want = _plain.linear_grad(y[rows], x[rows], s["weight"], pre[rows], "relu")
    _plain.within(dx[rows], want[0], want[1], "dx")
    _lib.device_status()


@pytest.mark.parametrize("m,k,n", [(2, 320, 640), (300, 320, 640), (300, 321, 643), (2500, 48, 40), (70, 3001, 24)])
def test_same_bits_every_time_and_from_graphs(m, k, n):
    """Two captured graphs, replayed in turn on a stream of their own with new inputs, give what eager calls give."""
    cuda_or_skip()
    _, ops = _ops()
    sets = [list(_inputs(m, k, n, torch.bfloat16, seed=s).values()) for s in (1, 2, 3)]

    def step(x, w, b, r, dy):
        y, pre = ops.linear_act(x, w, b, activation="gelu", residual=r, want_pre=True)
        return (y, pre, *ops.linear_act_bwd(dy, x, w, pre, "gelu"))

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
        for i in (2, 0, 1):
            for g, held, _ in graphs:
                for t, v in zip(held, sets[i]):
                    t.copy_(v)
                g.replay()
            side.synchronize()
            for _, _, got in graphs:
                assert all(torch.equal(p, q) for p, q in zip(got, want[i]))


def test_feed_forward_block_trains():
    """LayerNorm -> linear + gelu -> linear + residual, forward and backward with these operators alone, against autograd in 64
    bits.  Every stored intermediate is rounded to bf16, half a step (2^-8) at most: the results' relative 2-norm errors
    add up over the stages that a gradient has passed (y 4; gradients of the second layer 4, of the first 7, of the norm 9)."""
    cuda_or_skip()
    _lib, ops = _ops()
    m, c, f = 154, 640, 2560
    g = torch.Generator(device="cuda").manual_seed(0)
    rn = lambda *s, scale=1.0: (torch.randn(*s, device="cuda", generator=g) * scale).bfloat16()
    x, gamma, beta = rn(2, 77, c), rn(c, scale=0.2) + 1, rn(c, scale=0.2)
    w1, b1, w2, b2, dy = rn(f, c, scale=c**-0.5), rn(f, scale=0.2), rn(c, f, scale=f**-0.5), rn(c, scale=0.2), rn(2, 77, c)
    h, mean, rstd = ops.layernorm_fwd(x, gamma, beta, 1e-5, want_stats=True)
    u, pre = ops.linear_act(h, w1, b1, activation="gelu", want_pre=True)
    y = ops.linear_act(u, w2, b2, residual=x)
    du, dw2, db2 = ops.linear_act_bwd(dy, u, w2)
    dh, dw1, db1 = ops.linear_act_bwd(du, h, w1, pre, activation="gelu")
    dx, dgamma, dbeta = ops.layernorm_bwd(dh, x, mean, rstd, gamma)
    dx = dx.float() + dy.float()
    _lib.device_status()
    leaves = [t.double().requires_grad_() for t in (x, gamma, beta, w1, b1, w2, b2)]
    fn = torch.nn.functional
    ref = leaves[0] + fn.linear(fn.gelu(fn.linear(fn.layer_norm(leaves[0], (c,), leaves[1], leaves[2], 1e-5), leaves[3], leaves[4])), leaves[5], leaves[6])
    want = torch.autograd.grad(ref, leaves, dy.double())
    for got, ref, stages, what in [(y, ref, 4, "y"), (dw2, want[5], 4, "dw2"), (db2, want[6], 1, "db2"), (dw1, want[3], 7, "dw1"), (db1, want[4], 7, "db1"),
                                   (dgamma, want[1], 9, "dgamma"), (dbeta, want[2], 9, "dbeta"), (dx, want[0], 9, "dx")]:
        off = float((got.double() - ref).norm() / ref.norm())
        assert off <= stages * 2.0**-8, f"{what}: {off:.2e}"


def test_counted_launches():
    """One kernel, one more for operands that the copy engine cannot read, none without rows."""
    cuda_or_skip()
    _lib, ops = _ops()

    def count(call):
        before = _lib.launches
        call()
        return _lib.launches - before

    s = _inputs(300, 64, 96, torch.float16)
    w, x, pre = s["weight"], s["x"], s["dy"]
    odd = torch.zeros(300, 65, device="cuda", dtype=torch.float16)[:, 1:]
    assert count(lambda: ops.linear_act(x, w)) == 1 and count(lambda: ops.linear_act(odd, w)) == 2 and count(lambda: ops.linear_act(x[:2], w)) == 1
    assert count(lambda: ops.linear_act(x[:0], w)) == 0 and count(lambda: ops.linear_act_bwd(s["dy"][:0], x[:0], w)) == 0
    assert count(lambda: ops.linear_act_bwd(s["dy"], x, w, pre, "gelu")) == 3     # dz, its sums, both products
    assert count(lambda: ops.linear_act_bwd(s["dy"], x, w, want_dbias=False)) == 1
    assert count(lambda: ops.linear_act_bwd(s["dy"], x, w, want_dbias=False, want_dx=False)) == 1
    assert count(lambda: ops.linear_act_bwd(s["dy"][:9], x[:9], w, pre[:9], "gelu")) == 2
    long = _inputs(9000, 64, 96, torch.float16)                                   # and one that joins parts of the long sum
    assert count(lambda: ops.linear_act_bwd(long["dy"], long["x"], long["weight"], want_dbias=False)) == 2
    big = _inputs(3000, 1280, 1280, torch.float16)                                # more tiles than SMs: two launches
    assert count(lambda: ops.linear_act_bwd(big["dy"], big["x"], big["weight"], want_dbias=False)) == 2
    n = torch.ones(64, device="cuda", dtype=torch.float16)
    rows = torch.zeros(2000, 64, device="cuda", dtype=torch.float16)
    _, mean, rstd = ops.layernorm_fwd(rows, n, want_stats=True)
    assert count(lambda: ops.layernorm_fwd(rows, n)) == 1 and count(lambda: ops.layernorm_fwd(rows[:0], n)) == 0
    assert count(lambda: ops.layernorm_bwd(rows, rows, mean, rstd, n)) == 2 and count(lambda: ops.layernorm_bwd(rows[:5], rows[:5], mean[:5], rstd[:5], n)) == 1


def test_mixed_devices_are_refused():
    cuda_or_skip()
    _, ops = _ops()
    x, w = torch.zeros(4, 8, device="cuda", dtype=torch.float16), torch.zeros(6, 8, device="cuda", dtype=torch.float16)
    mean = torch.zeros(4, device="cuda")
    for call in (lambda: ops.linear_act(x, w.cpu()), lambda: ops.linear_act(x, w, w[:, 0].contiguous().cpu()), lambda: ops.linear_act(x.cpu(), w), lambda: ops.layernorm_fwd(x, x[0].cpu()),
                 lambda: ops.layernorm_bwd(x.cpu(), x, mean, mean), lambda: ops.layernorm_bwd(x, x, mean.cpu(), mean), lambda: ops.linear_act_bwd(x[:, :6], x, w, out_of(x), "gelu")):
        with pytest.raises(ValueError, match="cuda|current CUDA device"):
            call()


def out_of(x):
    return torch.zeros(x.shape[0], 6, dtype=x.dtype)


def test_out_has_a_new_version():
    """What is written into ``out`` counts as a change: autograd refuses a graph that needs the values before, and cross-attention projects
    its conditioning again."""
    cuda_or_skip()
    _, ops = _ops()
    from basedxl_b200.layers import Attention

    x, w = _inputs(77, 64, 64, torch.float16)["x"][None], _inputs(1, 64, 64, torch.float16, 3)["weight"]
    calls = (lambda out: ops.layernorm_fwd(x, out=out), lambda out: ops.linear_act(x, w, out=out))
    for call in calls:
        out = x.clone()
        leaf = torch.ones_like(out).requires_grad_()
        product = leaf * out
        call(out)
        assert out._version == 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            product.sum().backward()
        with torch.inference_mode():
            call(torch.empty_like(x))
    assert ops.layernorm_fwd(x[:, :0], out=torch.empty_like(x)[:, :0])._version == 0

    layer = Attention(128, 2, 64).half().cuda()   # its context is 64 wide
    for call in calls:
        ctx = x.clone()
        with torch.no_grad():
            first = layer.context_kv(ctx).clone()
            call(ctx)
            kv = layer.context_kv(ctx).clone()
            assert not torch.equal(kv, first) and torch.equal(kv, layer.context_kv(ctx.clone()))
