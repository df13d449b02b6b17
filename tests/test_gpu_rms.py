"""Root-mean-square norm on the GPU against float64: output, the sum with a residual, the
gradients, and the microscaled output, over dtypes, widths on both sides of every layout
the kernels choose, rows from none to many, strides and alignments.

Tolerances, with u = 2^-24 and n the longest chain of additions behind one sum (n = 64 up to rows that registers
hold: at most 16 elements in a thread, 10 lane and wave steps; wide rows width / 1024 more):

* a sum of squares is off by n u of itself, r so by less than n u r, h = s r by dh = n u |h|, y = h w by |w| dh + 2 u |y|;
* dx = r (g - h c) + dsum, c = mean(g h): c is off by n u mean|g h| + mean(|g| dh), so dx by r (n u |g| + |h| (n u
  mean|g h| + mean(|g| dh)) + |c| dh) + n u |r (g - h c)| and 2 u of the last sum's terms;
* dw by sum |dy| (dh + rows u |h|);
* each result by half a step of its own dtype more: 2^-8 (bfloat16), 2^-11 (float16) or 2^-24 of its value.

The microscaled values lie between those of the exact norm less and plus its error: rounding does not
change an order.
"""
import pytest

torch = pytest.importorskip("torch")

import mx_reference as mx  # noqa: E402

pytestmark = pytest.mark.gpu

TDT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
U = 2.0 ** -24
TINY = 2.0 ** -25  # float16 below its normal range: half of its smallest step


@pytest.fixture(scope="module", autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def reference(x, w, res, dy, ds, eps, n):
    """float64 (y, dx, dw) and the bound of each one's error before its last rounding, and the sum as it is kept"""
    s = x if res is None else (x.float() + res.float()).to(x.dtype)
    v, dy = s.double(), dy.double()
    w = torch.ones(v.shape[-1], dtype=torch.float64) if w is None else w.double()
    r = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    h = v * r
    dh = n * U * h.abs()
    g = dy * w
    c = (g * h).mean(-1, keepdim=True)
    dx = r * (g - h * c)
    e_dx = r * (n * U * g.abs() + h.abs() * (n * U * (g * h).abs().mean(-1, keepdim=True)
                                             + (g.abs() * dh).mean(-1, keepdim=True)) + c.abs() * dh) + n * U * dx.abs()
    if ds is not None:
        e_dx = e_dx + 2 * U * (dx.abs() + ds.double().abs())
        dx = dx + ds.double()
    rows = n + x.shape[0] // 256
    return ((h * w, w.abs() * dh + 2 * U * (h * w).abs()), (dx, e_dx),
            ((dy * h).sum(0), (dy.abs() * (dh + rows * U * h.abs())).sum(0)), s)


def check(got, ref, name):
    want, bound = ref
    assert got.shape == want.shape, name
    tiny = TINY if got.dtype == torch.float16 else 0.0
    err = (got.double().cpu() - want).abs()
    tol = bound + STEP[got.dtype] * want.abs() * (1 + 2 ** -7) + tiny + 1e-37
    assert not bool((~(err <= tol)).any()), (name, float((err / tol).max()))


def make(rows, D, dt, seed, params=None, residual=True):
    gen = torch.Generator().manual_seed(seed)
    t = TDT[dt]
    x, res = ((torch.randn(rows, D, generator=gen) * s).to(t) for s in (1.0, 3.0))
    w = (1 + 0.2 * torch.randn(D, generator=gen)).to(TDT[params or dt])
    dy, ds = (torch.randn(rows, D, generator=gen).to(t) for _ in range(2))
    return (x, w, res, dy, ds) if residual else (x, w, None, dy, None)


def run(x, w, res, dy, ds, eps=1e-6):
    """y, s (x without a residual), dx, dres (dx without), dw"""
    from mask_loss_amd.functions import rms_norm
    leaves = [None if t is None else t.cuda().requires_grad_(True) for t in (x, w, res)]
    out = rms_norm(leaves[0], leaves[1], eps, leaves[2])
    if res is None:
        g = torch.autograd.grad(out, leaves[:2], dy.cuda())
        return out.detach(), leaves[0].detach(), g[0], g[0], g[1]
    g = torch.autograd.grad(out, leaves, (dy.cuda(), ds.cuda()))
    return out[0].detach(), out[1].detach(), g[0], g[2], g[1]


def compare(args, n=64, eps=1e-6):
    got, ref = run(*args, eps=eps), reference(*args, eps, n)
    assert torch.equal(got[1].cpu(), ref[3])
    for g, r, name in zip((got[0], got[2], got[3], got[4]), (ref[0], ref[1], ref[1], ref[2]), ("y", "dx", "dres", "dw")):
        check(g, r, name)


# widths around every choice of threads and vectors: 16, 32 and 64 lanes, a
# workgroup of 256 and of 1024, rows that registers do not hold, odd ones
WIDTHS = [1, 2, 7, 31, 64, 100, 128, 129, 255, 256, 257, 512, 520, 1000, 1024, 1025, 1153, 2048, 2056, 4096, 4104, 8192,
          8193, 8200, 20000]


@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", WIDTHS)
def test_widths(dt, D, residual):
    compare(make(37 if D < 2500 else 9, D, dt, D, residual=residual))


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,D", [(1, 256), (2, 64), (3, 4096), (5, 8192), (1, 20000), (4097, 256), (20011, 96),
                                    (2600, 1153), (3001, 2048)])
def test_rows(dt, rows, D):
    compare(make(rows, D, dt, rows))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("D", [200, 4096, 9000])
def test_float32_weight(dt, D):
    args = make(50, D, dt, 3, params="f32")
    compare(args)
    assert run(*args)[4].dtype == torch.float32


@pytest.mark.parametrize("used", ["y", "sum", "both"])
def test_gradients_of_one_output(used):
    """One of the two outputs used, and each leaf alone."""
    from mask_loss_amd.functions import rms_norm
    x, w, res, dy, ds = make(33, 320, "bf16", 4)
    zero = torch.zeros_like(dy)
    ref = reference(x, w, res, dy if used != "sum" else zero, ds if used != "y" else None, 1e-6, 64)
    for want in range(3):
        leaves = [t.cuda() for t in (x, w, res)]
        leaves[want].requires_grad_(True)
        y, s = rms_norm(leaves[0], leaves[1], 1e-6, leaves[2])
        outs = {"y": (y,), "sum": (s,), "both": (y, s)}[used]
        ups = {"y": (dy.cuda(),), "sum": (ds.cuda(),), "both": (dy.cuda(), ds.cuda())}[used]
        g, = torch.autograd.grad(outs, leaves[want], ups, allow_unused=used == "sum" and want == 1)
        check(g, ref[2] if want == 1 else ref[1], "gradient %d" % want)


def test_input_is_its_own_residual():
    """The same tensor twice: the gradients of both places add up."""
    from mask_loss_amd.functions import rms_norm
    x, w, _, dy, ds = make(20, 96, "f32", 5)
    leaf = x.cuda().requires_grad_(True)
    y, s = rms_norm(leaf, w.cuda(), 1e-6, leaf)
    g, = torch.autograd.grad((y, s), leaf, (dy.cuda(), ds.cuda()))
    (v, bound), ref = reference(x, w, x, dy, ds, 1e-6, 64)[1], None
    check(g, (2 * v, 2 * bound), "dx")


def test_no_rows_no_weight():
    from mask_loss_amd.functions import rms_norm, rms_norm_mx
    x = torch.zeros(0, 3, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y, s = rms_norm(x, w, residual=torch.zeros_like(x))
    gx, gw = torch.autograd.grad((y, s), (x, w), (torch.zeros_like(y), torch.zeros_like(s)))
    assert y.shape == s.shape == gx.shape == x.shape and not gw.any()
    codes, scales = rms_norm_mx(x.detach(), w.detach())
    assert codes.shape == x.shape and scales.shape == (0, 3, 2)
    args = make(33, 200, "bf16", 6)
    ref = reference(args[0], None, *args[2:], 1e-6, 64)
    leaf = args[0].cuda().requires_grad_(True)
    y, s = rms_norm(leaf, residual=args[2].cuda())
    check(y.detach(), ref[0], "y")
    g, = torch.autograd.grad((y, s), leaf, (args[3].cuda(), args[4].cuda()))
    check(g, ref[1], "dx")


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_layouts(dt):
    """Tensors of four dimensions, transposed ones, rows on no 16-byte boundary, and upstream gradients that are
    broadcast."""
    from mask_loss_amd.functions import rms_norm, rms_norm_mx
    x, w, res, _, _ = make(30, 256, dt, 7)
    ones = torch.ones(30, 256)
    x4, r4 = x.view(2, 3, 5, 256).transpose(0, 2), res.view(5, 3, 2, 256)
    flat = lambda t: t.reshape(-1, 256)  # noqa: E731
    ref = reference(flat(x4), w, flat(r4), ones, ones, 1e-6, 64)
    leaf, other = x4.cuda().requires_grad_(True), r4.cuda().requires_grad_(True)
    y, s = rms_norm(leaf, w.cuda(), 1e-6, other)
    assert y.shape == s.shape == x4.shape
    (y.sum() + s.sum()).backward()
    check(flat(y.detach()), ref[0], "y")
    assert torch.equal(flat(s.detach()).cpu(), ref[3])
    check(flat(leaf.grad), ref[1], "dx")
    check(flat(other.grad), ref[1], "dres")
    room = torch.empty(30 * 256 + 1, dtype=TDT[dt], device="cuda")
    room[1:] = x.reshape(-1).cuda()
    off = room[1:].view(30, 256)
    assert off.data_ptr() % 16 != 0
    compare_to = reference(x, w, res, ones, None, 1e-6, 64)
    for a, b in ((off, res.cuda()), (x.cuda(), None)):
        if b is None:
            room[1:] = res.reshape(-1).cuda()
            b = off
        y, s = rms_norm(a, w.cuda(), 1e-6, b)
        check(y, compare_to[0], "y")
        leaf = a.clone().requires_grad_(True) if a is not off else off.detach().requires_grad_(True)
        g, = torch.autograd.grad(rms_norm(leaf, w.cuda(), 1e-6, b)[0].sum(), leaf)
        check(g, compare_to[1], "dx")
        got = rms_norm_mx(a, w.cuda(), 1e-6, b)
        want = rms_norm_mx(a.clone(), w.cuda(), 1e-6, b.clone())
        assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(got[:2], want[:2]))


@pytest.mark.parametrize("format", ["e4m3", "e2m1"])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,D,residual", [(1, 32, True), (37, 64, False), (5, 96, True), (19, 128, True), (33, 256, False),
                                             (9, 544, True), (40, 1024, True), (7, 2048, False), (11, 4128, True),
                                             (3, 8192, True), (3, 8224, True), (2, 20000, False), (3001, 256, True)])
def test_microscaled_output(format, dt, rows, D, residual):
    from mask_loss_amd.functions import rms_norm_mx
    x, w, res, dy, _ = make(rows, D, dt, 8, residual=residual)
    x[0] = 0  # rows of zeros without a residual
    (y, err), _, _, s = reference(x, w, res, dy, None, 1e-6, 64)
    out = rms_norm_mx(x.cuda(), w.cuda(), 1e-6, None if res is None else res.cuda(), format=format)
    codes, scales = out[:2]
    assert scales.shape == (rows, D // 32) and scales.dtype == torch.float8_e8m0fnu
    assert codes.shape == ((rows, D) if format == "e4m3" else (rows, D // 2))
    if res is not None:
        assert torch.equal(out[2].cpu(), s)
    b = mx.byte(scales)
    lo, hi = ((y.abs() + k * err).clamp_min(0) for k in (-1, 1))
    assert bool((b >= mx.scale_codes(lo, format)).all()) and bool((b <= mx.scale_codes(hi, format)).all())
    q = mx.values(codes)
    assert bool((q >= mx.nearest(mx.divide(y - err, b), format)).all())
    assert bool((q <= mx.nearest(mx.divide(y + err, b), format)).all())


def test_values():
    """Large and tiny rows, rows of zeros with and without eps, and a NaN or an infinity that stays in its row (and,
    quantised, in its blocks)."""
    from mask_loss_amd.functions import rms_norm, rms_norm_mx
    x, w, res, dy, ds = make(40, 256, "f32", 9)
    x[3], res[3] = 0.0, 0.0
    x[4] *= 2.0 ** 40
    x[5], res[5] = x[5] * 2.0 ** -40, 0.0
    compare((x, w, res, dy, ds))
    zero = torch.zeros(2, 64, device="cuda")
    assert not rms_norm(zero).any()
    assert torch.isnan(rms_norm(zero, eps=0.0)).all()  # 0 / 0
    bad = x.clone()
    bad[7, 3], bad[9, 0] = float("nan"), float("inf")
    keep = [i for i in range(40) if i not in (7, 9)]
    y, clean = (rms_norm(t.cuda(), w.cuda()).cpu() for t in (bad, x))
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[7]).all() and torch.isnan(y[9, 0])
    (c1, s1), (c2, s2) = (rms_norm_mx(t.cuda(), w.cuda()) for t in (bad, x))
    assert torch.equal(c1[keep].view(torch.uint8), c2[keep].view(torch.uint8)) and torch.equal(mx.byte(s1)[keep], mx.byte(s2)[keep])
    assert bool((mx.byte(s1)[7] == 255).all()) and int(mx.byte(s1)[9, 0]) == 255


def test_gradient_against_differences():
    x, w, res, dy, ds = make(20, 160, "f32", 10)

    def loss(x, w, res):
        s = x + res
        return float((s / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-6) * w * dy.double()).sum() + (s * ds.double()).sum())

    _, _, gx, gr, gw = run(x, w, res, dy, ds)
    gen = torch.Generator().manual_seed(11)
    args = [t.double() for t in (x, w, res)]
    step = 1e-4
    for i, g in enumerate((gx, gw, gr)):
        v = torch.randn(args[i].shape, generator=gen, dtype=torch.float64)
        hi, lo = ([t + k * step * v if j == i else t for j, t in enumerate(args)] for k in (1, -1))
        want = (loss(*hi) - loss(*lo)) / (2 * step)
        got = float((g.double().cpu() * v).sum())
        # third derivatives times step^2, and float32 gradients: both below 1e-5 of the sum's size
        assert abs(got - want) <= 1e-5 * float((g.double().cpu() * v).abs().sum()) + 1e-7, i


def test_widest():
    """A width of 2^26, the most that the norm takes: a thread adds width / 1024 terms."""
    D = 1 << 26
    gen = torch.Generator(device="cuda").manual_seed(12)
    x, res, dy, ds = (torch.randn(2, D, generator=gen, device="cuda").bfloat16() for _ in range(4))
    w = (1 + 0.2 * torch.randn(D, generator=gen, device="cuda")).bfloat16()
    got = run(x, w, res, dy, ds)
    ref = reference(x, w.double(), res, dy, ds, 1e-6, 64 + D // 1024)
    assert torch.equal(got[1], ref[3])
    for g, (v, bound), name in zip((got[0], got[2], got[4]), ref[:3], ("y", "dx", "dw")):
        assert bool(((g.double() - v).abs() <= bound + 2.0 ** -8 * v.abs() * (1 + 2 ** -7) + 1e-37).all()), name


def test_rows_past_32_bits():
    """4.3e9 elements: the last rows as in a call of their own."""
    from mask_loss_amd.functions import rms_norm, rms_norm_mx
    R, D, n = (1 << 22) + 100, 1056, 50
    xs, w, rs, _, _ = make(n, D, "bf16", 13)
    few = rms_norm(xs.cuda(), w.cuda(), 1e-6, rs.cuda())
    x = torch.zeros(R, D, dtype=torch.bfloat16, device="cuda")
    res = torch.zeros(R, D, dtype=torch.bfloat16, device="cuda")
    x[-n:], res[-n:] = xs.cuda(), rs.cuda()
    y, s = rms_norm(x, w.cuda(), 1e-6, res)
    assert torch.equal(y[-n:], few[0]) and torch.equal(s[-n:], few[1]) and not bool(y[:-n].any())
    del y, s
    codes, scales, _ = rms_norm_mx(x, w.cuda(), 1e-6, res)
    c, b, _ = rms_norm_mx(xs.cuda(), w.cuda(), 1e-6, rs.cuda())
    assert torch.equal(codes[-n:].view(torch.uint8), c.view(torch.uint8)) and torch.equal(mx.byte(scales[-n:]), mx.byte(b))


def test_refusals():
    from mask_loss_amd.functions import rms_norm, rms_norm_mx
    x, w = torch.zeros(4, 64, device="cuda"), torch.ones(64, device="cuda")
    bad = [(x.double(), None, None, "float32, bfloat16 or float16"), (x.half(), w.bfloat16(), None, "input's dtype"),
           (x, w[:32], None, "shape"), (x, w.cpu(), None, "CUDA tensor"), (x[:, :0], None, None, "at least 1"),
           (x, None, x[:3], "residual must match"), (x, None, x.half(), "residual must match"), (x, None, x.cpu(), "CUDA tensor")]
    for x_, w_, r_, words in bad:
        for grad in (False, True):
            with pytest.raises(RuntimeError, match=words):
                rms_norm(x_.detach().requires_grad_(grad), w_, 1e-6, r_)
        with pytest.raises(RuntimeError, match=words):
            rms_norm_mx(x_, w_, 1e-6, r_)
    for eps in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            rms_norm(x, w, eps)
        with pytest.raises(ValueError, match="eps"):
            rms_norm_mx(x, w, eps)
    with pytest.raises(RuntimeError, match="multiple of 32"):
        rms_norm_mx(x[:, :48], None)
    with pytest.raises(NotImplementedError, match="no gradient"):
        rms_norm_mx(x, w.clone().requires_grad_(True))
