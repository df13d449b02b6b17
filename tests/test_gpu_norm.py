"""Layer norm on the GPU against float64: output and the gradients of input,
weight and bias, over dtypes, widths on both sides of every layout the kernels
choose, rows from none to many, strides, alignments and streams.

Tolerances, with u = 2^-24 the rounding of float32 and n the longest chain of
additions behind one sum (at most 8 vectors' elements in a thread, 10 lane and
wave steps, for wide rows width / 1024 in a thread, for the weights' gradients
their rows; 64 covers the first three here):

* the mean is off by n u max|x|, the normalised value h = (x - m) r so by
  dh = n u (max|x| r + |h|), and y = h w + b by |w| dh + 2 u (|h w| + |y|);
* dx = r (g - mean g - h c), c = mean(g h), by r times n u (|g| + mean|g| + 2 |h|
  mean|g h|) + |c| dh + |h| mean(|g| dh);
* dw by sum |dy| (dh + n u |h|), db by n u sum |dy|;
* each result by half a step of its own dtype more: 2^-8 (bfloat16), 2^-11
  (float16) or 2^-24 of its value.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TDT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
U = 2.0 ** -24
TINY = 2.0 ** -25  # float16 below its normal range: half of its smallest step


@pytest.fixture(scope="module", autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def reference(x, w, b, dy, eps, n):
    """float64 (y, dx, dw, db) and the bound of each one's error before its last rounding"""
    x, dy = x.double(), dy.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(x.shape[-1], dtype=torch.float64) if b is None else b.double()
    m = x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + eps)
    h = (x - m) * r
    y = h * w + b
    dh = n * U * (x.abs().amax(-1, keepdim=True) * r + h.abs())
    g = dy * w
    c = (g * h).mean(-1, keepdim=True)
    dx = r * (g - g.mean(-1, keepdim=True) - h * c)
    e_dx = r * (n * U * (g.abs() + g.abs().mean(-1, keepdim=True) + 2 * h.abs() * (g * h).abs().mean(-1, keepdim=True))
                + c.abs() * dh + h.abs() * (g.abs() * dh).mean(-1, keepdim=True))
    rows = n + x.shape[0] // 256
    return ((y, w.abs() * dh + 2 * U * ((h * w).abs() + y.abs())), (dx, e_dx),
            ((dy * h).sum(0), (dy.abs() * (dh + rows * U * h.abs())).sum(0)), (dy.sum(0), rows * U * dy.abs().sum(0)))


def check(got, ref, name):
    want, bound = ref
    assert got.shape == want.shape, name
    tiny = TINY if got.dtype == torch.float16 else 0.0
    err = (got.double().cpu() - want).abs()
    tol = bound + STEP[got.dtype] * want.abs() * (1 + 2 ** -7) + tiny + 1e-37
    bad = ~(err <= tol)
    assert not bool(bad.any()), (name, float((err / tol).max()))


def make(rows, D, dt, seed, params=None, shift=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, D, generator=gen) + shift * torch.randn(D, generator=gen)).to(TDT[dt])
    p = TDT[params or dt]
    w = (1 + 0.2 * torch.randn(D, generator=gen)).to(p)
    b = (0.2 * torch.randn(D, generator=gen)).to(p)
    dy = torch.randn(rows, D, generator=gen).to(TDT[dt])
    return x, w, b, dy


def run(x, w, b, dy, eps=1e-5):
    from mask_loss_amd.functions import layer_norm
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves, eps)
    return (y.detach(), *torch.autograd.grad(y, leaves, dy.cuda()))


# widths around every choice of threads and vectors: 16, 32 and 64 lanes, a
# workgroup of 256 and of 1024, rows that registers do not hold, odd ones
WIDTHS = [1, 2, 7, 31, 64, 100, 128, 129, 255, 256, 257, 384, 512, 520, 768, 1000, 1024, 1025, 1153, 2048, 2056, 4096,
          4104, 5000, 8192, 8193, 8200, 20000]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", WIDTHS)
def test_widths(dt, D):
    rows = 37 if D < 3000 else 9
    x, w, b, dy = make(rows, D, dt, D)
    for got, ref, name in zip(run(x, w, b, dy), reference(x, w, b, dy, 1e-5, 64), ("y", "dx", "dw", "db")):
        check(got, ref, name)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,D", [(1, 256), (2, 64), (3, 4096), (5, 8192), (1, 20000), (4097, 256), (20011, 96),
                                    (2600, 1153), (3001, 2048)])
def test_rows(dt, rows, D):
    x, w, b, dy = make(rows, D, dt, rows)
    for got, ref, name in zip(run(x, w, b, dy), reference(x, w, b, dy, 1e-5, 64), ("y", "dx", "dw", "db")):
        check(got, ref, name)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D", [200, 256, 4096, 9000])
def test_float32_parameters(dt, D):
    x, w, b, dy = make(50, D, dt, 3, params="f32")
    got = run(x, w, b, dy)
    assert [t.dtype for t in got] == [TDT[dt], TDT[dt], torch.float32, torch.float32]
    for g, ref, name in zip(got, reference(x, w, b, dy, 1e-5, 64), ("y", "dx", "dw", "db")):
        check(g, ref, name)


@pytest.mark.parametrize("which", ["none", "weight", "bias"])
@pytest.mark.parametrize("params", ["f32", "bf16"])
def test_optional_parameters_and_gradients(which, params):
    from mask_loss_amd.functions import layer_norm
    x, w, b, dy = make(33, 320, "bf16", 4, params=params)
    w, b = (w if which == "weight" else None), (b if which == "bias" else None)
    dev = [None if t is None else t.cuda() for t in (x, w, b)]
    ref = reference(x, w, b, dy, 1e-5, 64)
    check(layer_norm(*dev), ref[0], "y")  # no gradients wanted
    for want in (0, 1, 2):  # one leaf at a time
        if dev[want] is None:
            continue
        leaves = [None if t is None else t.clone() for t in dev]
        leaves[want].requires_grad_(True)
        y = layer_norm(*leaves)
        g, = torch.autograd.grad(y, leaves[want], dy.cuda())
        assert g.dtype == leaves[want].dtype
        check(y.detach(), ref[0], "y")
        check(g, ref[want + 1], "gradient %d" % want)


def test_no_rows():
    from mask_loss_amd.functions import layer_norm
    x = torch.zeros(0, 3, 24, device="cuda", requires_grad=True)
    w = torch.ones(24, device="cuda", requires_grad=True)
    b = torch.ones(24, device="cuda", requires_grad=True)
    y = layer_norm(x, w, b)
    assert y.shape == x.shape
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
    assert gx.shape == x.shape and not gw.any() and not gb.any()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_layouts(dt):
    """A query tensor of four dimensions, a transposed one, rows on no 16-byte
    boundary, and an upstream gradient that is broadcast."""
    from mask_loss_amd.functions import layer_norm
    x, w, b, _ = make(6 * 5, 256, dt, 5)
    ref = lambda x, dy: reference(x.reshape(-1, 256), w, b, dy.reshape(-1, 256), 1e-5, 64)  # noqa: E731
    x4 = x.view(2, 3, 5, 256)
    ones = torch.ones(30, 256)
    for t, want in ((x4, x4), (x4.transpose(0, 2), x4.transpose(0, 2))):
        leaf = t.cuda().requires_grad_(True)
        y = layer_norm(leaf, w.cuda(), b.cuda())
        assert y.shape == want.shape
        y.sum().backward()
        check(y.detach().reshape(-1, 256), ref(want, ones)[0], "y")
        check(leaf.grad.reshape(-1, 256), ref(want, ones)[1], "dx")
    flat = torch.empty(30 * 256 + 1, dtype=TDT[dt], device="cuda")
    flat[1:] = x.reshape(-1).cuda()
    off = flat[1:].view(30, 256)
    assert off.data_ptr() % 16 != 0
    check(layer_norm(off, w.cuda(), b.cuda()), ref(x, ones)[0], "y")
    leaf = off.detach().requires_grad_(True)
    gx, = torch.autograd.grad(layer_norm(leaf, w.cuda(), b.cuda()).sum(), leaf)
    check(gx, ref(x, ones)[1], "dx")
    odd_w = torch.empty(257, dtype=TDT[dt], device="cuda")
    odd_w[1:] = w.cuda()
    check(layer_norm(x.cuda(), odd_w[1:], b.cuda()), ref(x, ones)[0], "y")
    big = torch.randn(30, 300).to(TDT[dt])
    check(layer_norm(big.cuda()[:, 10:266], w.cuda(), b.cuda()),
          ref(big[:, 10:266], ones)[0], "y")


def test_values():
    """Constant rows give the bias, a large common offset costs only its own rounding,
    and a NaN or an infinity stays in its row."""
    from mask_loss_amd.functions import layer_norm
    x, w, b, dy = make(40, 256, "f32", 6)
    x[3] = 7.0
    x[4] = 0.0
    got = run(x, w, b, dy)
    ref = reference(x, w, b, dy, 1e-5, 64)
    for g, r, name in zip(got, ref, ("y", "dx", "dw", "db")):
        check(g, r, name)
    assert torch.equal(got[0][4].cpu(), b)
    far, w, b, dy = make(40, 512, "f32", 7)
    far += 4096.0
    for g, r, name in zip(run(far, w, b, dy), reference(far, w, b, dy, 1e-5, 64), ("y", "dx", "dw", "db")):
        check(g, r, name)
    bad = x.clone()
    bad[7, 3], bad[9, 0] = float("nan"), float("inf")
    y = layer_norm(bad.cuda(), w[:256].cuda(), b[:256].cuda()).cpu()
    clean = layer_norm(x.cuda(), w[:256].cuda(), b[:256].cuda()).cpu()
    keep = [i for i in range(40) if i not in (7, 9)]
    assert torch.equal(y[keep], clean[keep])
    assert torch.isnan(y[[7, 9]]).all()


def test_gradient_against_differences():
    """The gradients along random directions against central differences of the
    float64 definition."""
    x, w, b, dy = make(20, 160, "f32", 8)

    def loss(x, w, b):
        m = x.mean(-1, keepdim=True)
        h = (x - m) / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + 1e-5)
        return float(((h * w + b) * dy.double()).sum())

    _, *grads = run(x, w, b, dy)
    gen = torch.Generator().manual_seed(9)
    args = [t.double() for t in (x, w, b)]
    step = 1e-4
    for i, g in enumerate(grads):
        v = torch.randn(args[i].shape, generator=gen, dtype=torch.float64)
        hi = [t + step * v if j == i else t for j, t in enumerate(args)]
        lo = [t - step * v if j == i else t for j, t in enumerate(args)]
        want = (loss(*hi) - loss(*lo)) / (2 * step)
        got = float((g.double().cpu() * v).sum())
        # third derivatives times step^2, and float32 gradients: both below 1e-5 of the sum's size
        scale = float((g.double().cpu() * v).abs().sum())
        assert abs(got - want) <= 1e-5 * scale + 1e-7, i


def test_runs_are_equal_and_streams():
    from mask_loss_amd.functions import layer_norm
    x, w, b, dy = make(5000, 256, "bf16", 10)
    first = run(x, w, b, dy)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, run(x, w, b, dy)))
    side = torch.cuda.Stream()
    xs, ws, bs = x.cuda(), w.cuda(), b.cuda()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = layer_norm(xs, ws, bs)
    side.synchronize()
    assert torch.equal(y, first[0])


def test_captured_step():
    from mask_loss_amd.functions import layer_norm
    x, w, b, dy = make(700, 256, "bf16", 11)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    dyd = dy.cuda()

    def step():
        y = layer_norm(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dyd))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in (12, 13, 14):
        x, _, _, dy = make(700, 256, "bf16", seed)
        with torch.no_grad():
            leaves[0].copy_(x)
            dyd.copy_(dy)
        graph.replay()
        torch.cuda.synchronize()
        want = run(x, w, b, dy)
        assert all(torch.equal(p, q) for p, q in zip(outs, want))


def test_refusals():
    from mask_loss_amd.functions import layer_norm
    x, w, b = torch.zeros(4, 64, device="cuda"), torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    bad = [(x.double(), None, None, "float32, bfloat16 or float16"), (x.half(), w.bfloat16(), None, "input's dtype"),
           (x.half(), w, b.half(), "same dtype"), (x, w[:32], None, "shape"), (x, None, b.view(1, 64), "shape"),
           (x, w.cpu(), None, "CUDA tensor"), (x[:, :0], None, None, "at least 1"),
           (torch.zeros((), device="cuda"), None, None, "at least 1")]
    for x_, w_, b_, words in bad:
        for grad in (False, True):
            with pytest.raises(RuntimeError, match=words):
                layer_norm(x_.detach().requires_grad_(grad), w_, b_)
    for eps in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            layer_norm(x, w, b, eps)


def test_second_derivative_is_refused():
    from mask_loss_amd.functions import layer_norm
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y = layer_norm(x, w)
    gx, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        gx.sum().backward()


def test_rows_past_32_bits():
    """4.3e9 elements: the last rows as in a call of their own, and the sums of their gradients."""
    from mask_loss_amd.functions import layer_norm
    R, D, n = (1 << 22) + 100, 1032, 50
    xs, w, b, dys = make(n, D, "bf16", 9)
    few = run(xs, w, b, dys)
    x = torch.zeros(R, D, dtype=torch.bfloat16, device="cuda")
    dy = torch.zeros(R, D, dtype=torch.bfloat16, device="cuda")
    x[-n:], dy[-n:] = xs.cuda(), dys.cuda()
    leaves = [x.requires_grad_(True), w.cuda().requires_grad_(True), b.cuda().requires_grad_(True)]
    y = layer_norm(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(y.detach()[-n:], few[0]) and torch.equal(dx[-n:], few[1])
    assert torch.equal(y.detach()[0], leaves[2].detach()) and not bool(dx[:-n].any())
    ref = reference(xs, w, b, dys, 1e-5, 64)  # (the other rows add zeros)
    check(dw, ref[2], "dw")
    check(db, ref[3], "db")
