"""Grouped products and mask logits on the GPU against float64: output and both
gradients, over dtypes, storage orders, ragged groups (empty ones, one row, rows in
no group), sizes on both sides of every tile, equal groups that share matrices.

Tolerance: products of 16-bit values are exact in float32 (float32 products round by
2^-24 each) and a sum of n of them is off by at most n 2^-24 sum |a b| in any order;
the result by half a step of its own dtype more (2^-8 bfloat16, 2^-11 float16,
2^-24 float32 of its value; 2^-25 below float16's normal range).
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TDT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def check(got, want, size, n, name):
    """size: sum |a b| of every element, n: its number of terms"""
    assert got.shape == want.shape, (name, got.shape, want.shape)
    err = (got.double().cpu() - want).abs()
    tol = ((n + 2) * U * size + STEP[got.dtype] * want.abs() * (1 + 2.0 ** -7)
           + (2.0 ** -25 if got.dtype == torch.float16 else 0.0) + 1e-37)
    bad = ~(err <= tol)
    assert not bool(bad.any()), (name, int(bad.sum()), float((err / tol).max()), bad.nonzero()[:4].tolist())


def edges_of(offsets, rows):
    """The groups' borders as the operator takes them."""
    e = np.maximum.accumulate(np.clip(np.asarray(offsets, dtype=np.int64), 0, rows))
    return [(int(lo), int(hi)) for lo, hi in zip(e, e[1:])]


def reference(x, w, dy, offsets, transposed):
    """float64 (value, size, terms) of y, dx and dw"""
    x, w, dy = x.double(), w.double(), dy.double()
    wm = w.transpose(1, 2) if transposed else w
    M, K, N = wm.shape
    outs = [[torch.zeros(x.shape[0], N).double(), torch.zeros_like(x), torch.zeros_like(wm)] for _ in range(2)]
    most = 0
    for g, (lo, hi) in enumerate(edges_of(offsets, x.shape[0])):
        for o, f in zip(outs, (lambda t: t, torch.abs)):
            o[0][lo:hi] = f(x[lo:hi]) @ f(wm[g % M])
            o[1][lo:hi] = f(dy[lo:hi]) @ f(wm[g % M]).T
            o[2][g % M] += f(x[lo:hi]).T @ f(dy[lo:hi])
        most += hi - lo
    if transposed:
        for o in outs:
            o[2] = o[2].transpose(1, 2)
    return [(v, s, n) for v, s, n in zip(*outs, (K, N, most))]


def run(x, w, dy, offsets, transposed):
    from mask_loss_amd.functions import grouped_matmul
    leaves = [x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)]
    o = None if offsets is None else torch.tensor(offsets, dtype=torch.int64).cuda()
    y = grouped_matmul(*leaves, o, transposed)
    return (y.detach(), *torch.autograd.grad(y, leaves, dy.cuda()))


def make(rows, K, N, M, dt, transposed, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, K, generator=gen).to(TDT[dt])
    w = (torch.randn(*((M, N, K) if transposed else (M, K, N)), generator=gen) * max(K, 1) ** -0.5).to(TDT[dt])
    dy = (torch.randn(rows, N, generator=gen) * 0.1).to(TDT[dt])
    return x, w, dy


def compare(x, w, dy, offsets, transposed):
    for got, ref, name in zip(run(x, w, dy, offsets, transposed), reference(x, w, dy, offsets, transposed),
                              ("y", "dx", "dw")):
        check(got, *ref, name)


def offsets_of(counts, first=0):
    return [first] + (first + np.cumsum(counts)).tolist()


# (rows per group, rows behind the last, K, N): tiles of 32 and 128 rows and 128 columns, steps
# of 64 and 32 reduced elements, odd lengths, one row, one column, groups with no row
SHAPES = [
    ([1], 0, 1, 1), ([3, 0, 2], 4, 5, 7), ([1, 1, 0, 1], 0, 64, 128), ([0, 0], 3, 16, 24), ([33], 0, 65, 129),
    ([40, 0, 130, 1], 5, 96, 136), ([128, 256], 0, 128, 256), ([129, 127, 0], 1, 200, 100), ([5, 60, 31], 0, 256, 1000),
    ([200, 200], 0, 256, 640), ([64] * 5, 0, 72, 392), ([2, 9, 4, 0, 7, 1, 3, 6], 2, 520, 264), ([300], 7, 33, 1025),
    ([17, 400], 0, 1, 130), ([70, 80], 0, 130, 1), ([257, 1], 0, 320, 257), ([12, 20], 0, 4096, 96),
    ([513, 90], 0, 512, 768),
]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_ragged(dt, transposed, case):
    counts, behind, K, N = SHAPES[case]
    x, w, dy = make(sum(counts) + behind, K, N, len(counts), dt, transposed, case)
    compare(x, w, dy, offsets_of(counts), transposed)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("transposed", [False, True])
def test_long_reductions(dt, transposed):
    """Few tiles and a long reduced axis: split and joined, in each product."""
    x, w, dy = make(45, 8192, 72, 2, dt, transposed, 30)  # forward
    compare(x, w, dy, [0, 20, 45], transposed)
    x, w, dy = make(210, 64, 9001, 2, dt, transposed, 31)  # input gradient
    compare(x, w, dy, [0, 100, 210], transposed)
    x, w, dy = make(5003, 40, 130, 1, dt, transposed, 32)  # weight gradient
    compare(x, w, dy, [0, 5003], transposed)
    x, w, dy = make(2100, 48, 64, 3, dt, transposed, 33)
    compare(x, w, dy, [4, 2000, 2000, 2090], transposed)
    # the same with rows of whole 16-byte chunks, one tile and a few
    x, w, dy = make(120, 8192, 64, 1, dt, transposed, 34)
    compare(x, w, dy, [0, 120], transposed)
    x, w, dy = make(390, 2056, 8192, 2, dt, transposed, 35)
    compare(x, w, dy, [5, 180, 385], transposed)
    x, w, dy = make(6000, 64, 128, 1, dt, transposed, 36)
    compare(x, w, dy, [0, 5990], transposed)


# (rows, K, N, groups, matrices) whose products take the tiles of 128 x 256 and 256 x 256, whole and in parts,
# with groups that share a matrix or not; the last one's d input leaves a round of 256 x 256 tiles an eighth full
LARGE = [(1500, 64, 4104, 5, 5), (1500, 64, 4104, 10, 5), (300, 5120, 512, 5, 5), (300, 512, 5120, 20, 5),
         (3000, 64, 4104, 5, 5), (3000, 64, 4104, 12, 3), (1100, 6400, 64, 3, 3), (1500, 64, 5120, 8, 2),
         (300, 264, 8240, 10, 5), (3000, 64, 5120, 4, 1), (300, 520, 4096, 10, 5), (16384, 1024, 4096, 16, 16)]


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("shape", LARGE)
def test_large_tiles(dt, transposed, shape):
    rows, K, N, G, M = shape
    counts = np.random.default_rng(rows + G).multinomial(rows - 3, np.ones(G) / G)
    x, w, dy = make(rows, K, N, M, dt, transposed, G)
    got = run(x, w, dy, offsets_of(counts, 1), transposed)
    with torch.device("cuda"):
        ref = reference(x.cuda(), w.cuda(), dy.cuda(), offsets_of(counts, 1), transposed)
    for g, (v, size, n), name in zip(got, ref, ("y", "dx", "dw")):
        check(g, v.cpu(), size.cpu(), n, name)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_many_groups(dt):
    rng = np.random.default_rng(0)
    for G, rows in ((63, 200), (64, 90), (65, 65), (200, 500), (1000, 700), (4000, 300)):
        counts = rng.multinomial(rows - 7, np.ones(G) / G)
        x, w, dy = make(rows, 24, 40, G, dt, True, G)
        compare(x, w, dy, offsets_of(counts, 3), True)


@pytest.mark.parametrize("offsets", [[2, 9, 30, 30, 41], [0, 30, 10, 50, 50], [-5, 20, 1 << 40, 3, 60], [60, 60, 60, 60, 60],
                                     [-(1 << 40), -1, 0, 0, 0]])
@pytest.mark.parametrize("transposed", [False, True])
def test_any_offsets(offsets, transposed):
    """Borders that leave rows in no group, that decrease, or that lie outside the
    tensor: held to the rows and to the border before."""
    x, w, dy = make(50, 64, 96, 4, "bf16", transposed, 40)
    compare(x, w, dy, offsets, transposed)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("L,M,n", [(1, 3, 20), (3, 2, 40), (10, 2, 100), (70, 1, 5), (4, 5, 1)])
def test_shared_matrices(dt, L, M, n):
    """Groups g, g + M, ... share a matrix, with and without offsets."""
    K, N = 64, 200
    x, w, dy = make(L * M * n, K, N, M, dt, False, L)
    offsets = [n * i for i in range(L * M + 1)]
    compare(x, w, dy, offsets, False)
    got = run(x.view(L * M, n, K), w, dy.view(L * M, n, N), None, False)
    for a, b in zip(got, run(x, w, dy, offsets, False)):
        assert torch.equal(a.reshape(b.shape), b)
    rng = np.random.default_rng(L)  # ragged sets of every layer
    counts = rng.integers(0, n + 1, size=L * M)
    compare(x, w, dy, offsets_of(counts, 1 if counts.sum() < L * M * n else 0), False)


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("G,M", [(33, 1), (1000, 1), (66, 2), (140, 2), (400, 4), (4000, 2)])
def test_many_groups_of_a_matrix(G, M, aligned):
    """More groups to a matrix than make tiles together, or one matrix for all: ragged, some
    empty, rows before the first and behind the last."""
    rng = np.random.default_rng(G)
    rows = 3 * G + 200
    counts = rng.multinomial(rows - 30, rng.dirichlet(np.ones(G)))
    K, N = (64, 136) if aligned else (45, 131)
    x, w, dy = make(rows, K, N, M, "bf16", False, G)
    compare(x, w, dy, offsets_of(counts, 11), False)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_parts_of_the_last_tiles(dt):
    """More tiles than the GPU holds at once and a long reduction: the last tiles are split, in
    every product and with ragged groups, shared matrices and rows in no group."""
    rng = np.random.default_rng(3)
    M, K, N = 2, 384, 2304
    counts = rng.integers(120, 300, size=3 * M)
    x, w, dy = make(int(counts.sum()) + 20, K, N, M, dt, False, 90)
    compare(x, w, dy, offsets_of(counts, 7), False)
    x, w, dy = make(4300, 1152, 2200, 1, dt, True, 91)
    compare(x, w, dy, [9, 4290], True)
    x, w, dy = make(2600, 1024, 2048, 1, dt, False, 92)  # the weight's gradient in few large tiles
    compare(x, w, dy, [3, 2590], False)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_other_rows_do_not_reach_a_group(dt):
    """NaN and infinity in one group's rows, in its matrix or in rows of no group stay
    where they belong."""
    counts = [40, 25, 70]
    x, w, dy = make(150, 96, 136, 3, dt, False, 50)
    offsets = offsets_of(counts, 4)
    want = reference(x, w, dy, offsets, False)
    x2, w2, dy2 = x.clone(), w.clone(), dy.clone()
    for t in (x2, dy2):
        t[:4] = float("nan")
        t[139:] = float("inf")
        t[44:69] = float("nan")  # group 1
    w2[1] = float("inf")
    y, dx, dw = run(x2, w2, dy2, offsets, False)
    keep = [i for i in range(150) if not 44 <= i < 69]
    check(y[keep], want[0][0][keep], want[0][1][keep], want[0][2], "y")
    check(dx[keep], want[1][0][keep], want[1][1][keep], want[1][2], "dx")
    check(dw[[0, 2]], want[2][0][[0, 2]], want[2][1][[0, 2]], want[2][2], "dw")
    assert torch.isnan(y[44:69]).all()


def test_no_rows_no_columns():
    from mask_loss_amd.functions import grouped_matmul
    o = torch.zeros(3, dtype=torch.int64, device="cuda")
    x, w, dy = make(0, 32, 48, 2, "bf16", False, 60)
    y, dx, dw = run(x, w, dy, [0, 0, 0], False)
    assert y.shape == (0, 48) and dx.shape == (0, 32) and not dw.any()
    x, w, dy = make(7, 0, 48, 2, "bf16", False, 61)  # an empty sum is zero
    y, dx, dw = run(x, w, dy, [0, 3, 7], False)
    assert y.shape == (7, 48) and not y.any() and dx.shape == (7, 0) and dw.shape == (2, 0, 48)
    x, w, dy = make(7, 32, 0, 2, "bf16", False, 62)
    y, dx, dw = run(x, w, dy, [0, 3, 7], False)
    assert y.shape == (7, 0) and not dx.any() and dw.shape == (2, 32, 0)
    assert grouped_matmul(torch.zeros(0, 4, device="cuda"), torch.zeros(2, 4, 5, device="cuda"), o).shape == (0, 5)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_layouts(dt):
    """Operands that are not contiguous, that start off a 16-byte boundary, and a
    broadcast upstream gradient."""
    from mask_loss_amd.functions import grouped_matmul
    x, w, dy = make(90, 64, 128, 2, dt, False, 70)
    offsets = [0, 50, 90]
    o = torch.tensor(offsets).cuda()
    ref = reference(x, w, torch.ones_like(dy), offsets, False)

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.reshape(-1).cuda()
        return flat[1:].view(t.shape)

    def strided(t):
        return t.cuda().transpose(-1, -2).contiguous().transpose(-1, -2)

    for form in (shifted, strided):
        leaves = [form(x).detach().requires_grad_(True), form(w).detach().requires_grad_(True)]
        y = grouped_matmul(*leaves, o)
        grads = torch.autograd.grad(y.sum(), leaves)
        for got, want, name in zip((y.detach(), *grads), ref, ("y", "dx", "dw")):
            check(got, *want, name)
    wide = torch.zeros(6, dtype=torch.int64, device="cuda")
    wide[::2] = o
    assert torch.equal(grouped_matmul(x.cuda(), w.cuda(), wide[::2]), grouped_matmul(x.cuda(), w.cuda(), o))


@pytest.mark.parametrize("leaf", [0, 1])
def test_one_gradient(leaf):
    from mask_loss_amd.functions import grouped_matmul
    x, w, dy = make(90, 64, 128, 2, "bf16", True, 71)
    args = [x.cuda(), w.cuda()]
    args[leaf].requires_grad_(True)
    y = grouped_matmul(*args, torch.tensor([0, 50, 90]).cuda(), transposed=True)
    g, = torch.autograd.grad(y, args[leaf], dy.cuda())
    check(g, *reference(x, w, dy, [0, 50, 90], True)[leaf + 1], "gradient")


def test_gradient_against_differences():
    """The product is linear in each operand, so differences of the float64 definition
    give its gradient along a direction without a truncation error."""
    x, w, dy = make(60, 40, 72, 3, "f32", False, 72)
    offsets = [2, 20, 20, 55]
    _, dx, dw = run(x, w, dy, offsets, False)

    def loss(x, w):
        return float(sum(((x[lo:hi] @ w[g]) * dy.double()[lo:hi]).sum() for g, (lo, hi) in enumerate(edges_of(offsets, 60))))

    gen = torch.Generator().manual_seed(1)
    for i, g in enumerate((dx, dw)):
        args = [x.double(), w.double()]
        v = torch.randn(args[i].shape, generator=gen, dtype=torch.float64)
        ends = []
        for sign in (1, -1):
            moved = list(args)
            moved[i] = args[i] + sign * v
            ends.append(loss(*moved))
        prod = g.double().cpu() * v
        assert abs(float(prod.sum()) - (ends[0] - ends[1]) / 2) <= 80 * U * 10 * float(prod.abs().sum())


def test_runs_are_equal_and_streams():
    from mask_loss_amd.functions import grouped_matmul
    x, w, dy = make(700, 256, 1024, 3, "bf16", False, 80)
    offsets = [0, 300, 310, 690]
    first = run(x, w, dy, offsets, False)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, run(x, w, dy, offsets, False)))
    args = x.cuda(), w.cuda(), torch.tensor(offsets).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = grouped_matmul(*args)
    side.synchronize()
    assert torch.equal(y, first[0])


def test_captured_step():
    """A step with split reductions, replayed with other rows, groups and matrices."""
    from mask_loss_amd.functions import grouped_matmul
    x, w, dy = make(150, 64, 4096, 3, "bf16", False, 81)
    leaves = [x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)]
    dyd, o = dy.cuda(), torch.tensor([0, 50, 100, 150]).cuda()

    def step():
        y = grouped_matmul(*leaves, o)
        return (y.detach(), *torch.autograd.grad(y, leaves, dyd))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed, offsets in ((82, [0, 1, 1, 140]), (83, [10, 70, 149, 150]), (84, [0, 0, 0, 0])):
        x, w, dy = make(150, 64, 4096, 3, "bf16", False, seed)
        with torch.no_grad():
            leaves[0].copy_(x)
            leaves[1].copy_(w)
            dyd.copy_(dy)
            o.copy_(torch.tensor(offsets))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(outs, run(x, w, dy, offsets, False)))


def test_refusals():
    from mask_loss_amd.functions import grouped_matmul, mask_logits
    x, w = torch.zeros(6, 8, device="cuda"), torch.zeros(2, 8, 3, device="cuda")
    o = torch.tensor([0, 2, 6]).cuda()
    bad = [(x, w.half(), o, False, "same dtype"), (x.double(), w.double(), o, False, "float32, bfloat16 or float16"),
           (x, w, o.int(), False, "int64"), (x, w, o.cpu(), False, "CUDA tensor"), (x, w.cpu(), o, False, "CUDA tensor"),
           (x, w, o, True, "must have 3 columns"), (x, w[0], o, False, "weight must be"),
           (x, w, torch.tensor([0, 2, 4, 6]).cuda(), False, "multiple"), (x, w[:0], o, False, "multiple"),
           (x, w, torch.tensor([0]).cuda(), False, "groups \\+ 1"), (x, w, None, False, "without offsets"),
           (x[None], w, o, False, "with offsets"), (x.view(3, 2, 8), w, None, False, "multiple")]
    for x_, w_, o_, t, words in bad:
        for grad in (False, True):
            with pytest.raises(RuntimeError, match=words):
                grouped_matmul(x_.detach().requires_grad_(grad), w_, o_, t)
    q, f = torch.zeros(1, 2, 3, 8, device="cuda"), torch.zeros(2, 8, 4, 4, device="cuda")
    with pytest.raises(RuntimeError, match="same dtype"):
        mask_logits(q, f.half())
    many = torch.zeros(4002, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="4000 groups"):
        grouped_matmul(x, w[:1], many)


def test_second_derivative_is_refused():
    from mask_loss_amd.functions import grouped_matmul
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    w = torch.randn(1, 64, 8, device="cuda", requires_grad=True)
    y = grouped_matmul(x, w, torch.tensor([0, 4]).cuda())
    gx, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        gx.sum().backward()


# ---- mask logits ------------------------------------------------------------------
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("L,B,Q,C,H,W", [(1, 2, 100, 64, 16, 24), (3, 2, 20, 32, 9, 13), (10, 1, 7, 256, 8, 8),
                                         (1, 1, 1, 16, 1, 1)])
def test_mask_logits(dt, L, B, Q, C, H, W):
    from mask_loss_amd.functions import mask_logits
    gen = torch.Generator().manual_seed(C)
    q = torch.randn(L, B, Q, C, generator=gen).to(TDT[dt])
    f = (torch.randn(B, C, H, W, generator=gen) * C ** -0.5).to(TDT[dt])
    dz = (torch.randn(L, B, Q, H, W, generator=gen) * 0.1).to(TDT[dt])
    leaves = [q.cuda().requires_grad_(True), f.cuda().requires_grad_(True)]
    z = mask_logits(*leaves)
    grads = torch.autograd.grad(z, leaves, dz.cuda())
    offsets = [Q * i for i in range(L * B + 1)]
    ref = reference(q.reshape(-1, C), f.flatten(2), dz.reshape(-1, H * W), offsets, False)
    for got, (v, s, n), shape, name in zip((z.detach(), *grads), ref, (dz.shape, q.shape, f.shape), ("z", "dq", "df")):
        check(got, v.reshape(shape), s.reshape(shape), n, name)
    # a ragged set per image, in a buffer with room behind the last
    counts = [(3 * b + 1) % (Q + 1) for b in range(B)]
    rows = q[0].reshape(-1, C)
    z = mask_logits(rows.cuda(), f.cuda(), torch.tensor(offsets_of(counts)).cuda())
    v, s, n = reference(rows, f.flatten(2), torch.zeros(B * Q, H * W), offsets_of(counts), False)[0]
    check(z, v.view(-1, H, W), s.view(-1, H, W), n, "ragged")


def test_mask_logits_empty():
    from mask_loss_amd.functions import mask_logits
    q = torch.zeros(2, 0, 5, 8, device="cuda", requires_grad=True)
    f = torch.zeros(0, 8, 4, 4, device="cuda", requires_grad=True)
    z = mask_logits(q, f)
    assert z.shape == (2, 0, 5, 4, 4)
    assert [g.shape for g in torch.autograd.grad(z.sum(), (q, f))] == [q.shape, f.shape]
    z = mask_logits(torch.zeros(1, 2, 0, 8, device="cuda"), torch.zeros(2, 8, 4, 4, device="cuda"))
    assert z.shape == (1, 2, 0, 4, 4)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_head_and_matching_together(dt):
    """Queries through norm and mask logits into the matching loss and back: the
    gradients of every leaf against float64, from the loss's own logit gradient."""
    from mask_loss_amd.functions import MaskMatchingFunction, layer_norm, mask_logits
    rng = np.random.default_rng(5)
    L, B, Q, C, H, W, G, K = 2, 2, 24, 64, 16, 16, 5, 7
    t = TDT[dt]
    q0 = torch.from_numpy(rng.normal(size=(L, B, Q, C))).to(t)
    w0 = torch.from_numpy(1 + 0.1 * rng.normal(size=C)).to(t)
    b0 = torch.from_numpy(0.1 * rng.normal(size=C)).to(t)
    f0 = torch.from_numpy(rng.normal(size=(B, C, H, W)) * 2 * C ** -0.5).to(t)
    tgt = torch.from_numpy(rng.integers(0, G + 1, size=(B, H, W))).cuda()
    cls_t = torch.full((B, G + 1), -1)
    cls_t[:, 1:] = torch.from_numpy(rng.integers(0, K - 1, size=(B, G)))
    zc = torch.from_numpy(rng.normal(size=(L, B, Q, K))).to(t).cuda().requires_grad_(True)
    q, w, b, f = (v.cuda().requires_grad_(True) for v in (q0, w0, b0, f0))
    h = layer_norm(q, w, b)
    h.retain_grad()
    z = mask_logits(h, f)
    z.retain_grad()
    _, _, m, d, c = MaskMatchingFunction.apply(z, tgt, zc, cls_t.cuda(), 1.0, 1.0, 1.0, 1.0, 0, 1.0, 0.05, True, 1e30,
                                               -1.0, True, False, 1, "global", 0.0, None, 0.0, None, K - 1, "softmax")
    scale = 1024.0
    ((m.sum() + d.sum() + c.sum()) * scale).backward()
    assert float(z.grad.abs().max()) > 0 and z.grad.shape == (L, B, Q, H, W)
    offsets = [Q * i for i in range(L * B + 1)]
    ref = reference(h.detach().cpu().reshape(-1, C), f0.flatten(2), z.grad.cpu().reshape(-1, H * W), offsets, False)
    for got, (v, s, n), name in zip((z.detach(), h.grad, f.grad), ref, ("z", "dh", "df")):
        check(got, v.reshape(got.shape), s.reshape(got.shape), n, name)
    # the norm's gradients from the product's: bounds of a norm's own test, loosely (n = 64)
    x64, g64 = q0.double().reshape(-1, C), h.grad.double().cpu().reshape(-1, C)
    mean = x64.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((x64 - mean) ** 2).mean(-1, keepdim=True) + 1e-5)
    hat = (x64 - mean) * r
    g = g64 * w0.double()
    dx = r * (g - g.mean(-1, keepdim=True) - hat * (g * hat).mean(-1, keepdim=True))
    for got, want, size in ((q.grad, dx, r * g.abs().sum(-1, keepdim=True) * (1 + hat.abs())),
                            (w.grad, (g64 * hat).sum(0), (g64 * hat).abs().sum(0)),
                            (b.grad, g64.sum(0), g64.abs().sum(0))):
        check(got.reshape(want.shape), want, size, 64, "norm")


# ---- offsets past 32 bits ---------------------------------------------------------
@pytest.mark.parametrize("K", [264, 265])
def test_rows_past_32_bits(K):
    """2.2e9 elements of input and d input, rows at both ends of them that are not zero."""
    from mask_loss_amd.functions import grouped_matmul
    R, N = (1 << 23) + 300, 16
    keep = torch.cat([torch.arange(5), torch.arange(R - 200, R)])
    xs, w, dys = make(205, K, N, 2, "bf16", False, 40)
    x = torch.zeros(R, K, dtype=torch.bfloat16, device="cuda")
    dy = torch.zeros(R, N, dtype=torch.bfloat16, device="cuda")
    x[keep.cuda()], dy[keep.cuda()] = xs.cuda(), dys.cuda()
    leaves = [x.requires_grad_(True), w.cuda().requires_grad_(True)]
    y = grouped_matmul(*leaves, torch.tensor([0, 5, R - 200, R - 100, R]).cuda())
    dx, dw = torch.autograd.grad(y, leaves, dy)
    ref = reference(xs, w, dys, [0, 5, 5, 105, 205], False)
    for got, r, name in zip((y.detach()[keep.cuda()], dx[keep.cuda()], dw), ref, ("y", "dx", "dw")):
        check(got, *r, name)
    assert not bool(y[5:R - 200].any()) and not bool(dx[5:R - 200].any())


def test_matrices_past_32_bits():
    """2.5e9 elements of weight and d weight, the last matrix in use."""
    from mask_loss_amd.functions import grouped_matmul
    M, K = 600, 2048
    x, w1, dy = make(6, K, K, 1, "bf16", False, 41)
    w = torch.zeros(M, K, K, dtype=torch.bfloat16, device="cuda")
    w[-1] = w1[0].cuda()
    offsets = torch.zeros(M + 1, dtype=torch.int64)
    offsets[-1] = 6
    leaves = [x.cuda().requires_grad_(True), w.requires_grad_(True)]
    y = grouped_matmul(*leaves, offsets.cuda())
    dx, dw = torch.autograd.grad(y, leaves, dy.cuda())
    ref = reference(x, w1, dy, [0, 6], False)
    for got, r, name in zip((y.detach(), dx, dw[-1:]), ref, ("y", "dx", "dw")):
        check(got, *r, name)
    assert not bool(dw[:-1].any())


def test_logits_past_32_bits():
    """2.2e9 logits of one image: the last queries' and the gradients from theirs."""
    from mask_loss_amd.functions import mask_logits
    Q, C, H, W, n = 33000, 16, 256, 256, 40
    q = torch.randn(Q, C, generator=torch.Generator().manual_seed(42)).bfloat16()
    _, f, dz = make(n, C, H * W, 1, "bf16", False, 43)
    leaves = [q.view(1, 1, Q, C).cuda().requires_grad_(True), f.view(1, C, H, W).cuda().requires_grad_(True)]
    z = mask_logits(*leaves)
    g = torch.zeros_like(z)
    g[0, 0, -n:] = dz.view(n, H, W).cuda()
    dq, df = torch.autograd.grad(z, leaves, g)
    (zv, zs, zn), (qv, qs, qn), (fv, fs, fn) = reference(q[-n:], f, dz, [0, n], False)
    check(z.detach()[0, 0, -n:].flatten(1), zv, zs, zn, "z")
    check(dq[0, 0, -n:], qv, qs, qn, "dq")
    check(df.flatten(2), fv, fs, fn, "df")
    assert not bool(dq[0, 0, :-n].any())
