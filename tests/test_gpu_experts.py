"""Rows by expert on the GPU: the order against numpy's stable sort, the rows there exactly, the sums back and
the gradients against float64.

Tolerances, with u = 2^-24: a sum of k products is off by (k + 1) u sum |w y|, the gradient of the weights, a
sum of D products of which a lane adds at most D / 16 and four to six lane steps follow, by (D / 16 + 8) u sum |dout y|, the rows'
gradient by u of its value; each result by half a step of its own dtype more.
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


def plan(ids, experts):
    """(order, slots, offsets) of an int64 array (T, k)"""
    flat = np.where((ids < 0) | (ids >= experts), experts, ids).reshape(-1)
    order = np.argsort(flat, kind="stable")
    slots = np.empty_like(order)
    slots[order] = np.arange(len(order))
    offsets = np.searchsorted(flat[order], np.arange(experts + 1), side="left")
    return order, slots.reshape(ids.shape), offsets


def numbers(tokens, k, experts, seed, kind="any"):
    rng = np.random.default_rng(seed)
    if kind == "same":
        return np.full((tokens, k), experts - 1)
    if kind == "few":  # two experts take nearly all
        return np.where(rng.random((tokens, k)) < 0.9, rng.integers(0, 2, (tokens, k)) % experts, rng.integers(0, experts, (tokens, k)))
    if kind == "dropped":
        return rng.integers(-3, experts + 3, (tokens, k))
    if kind == "none":
        return np.where(rng.random((tokens, k)) < 0.5, -1, experts)
    return rng.integers(0, experts, (tokens, k))


def sort(ids, experts):
    from mask_loss_amd.functions import sort_by_expert
    return sort_by_expert(torch.from_numpy(ids).cuda(), experts)


# one workgroup (up to 4,096 assignments and 1,023 experts) and several, whole and cut waves and chunks
@pytest.mark.parametrize("kind", ["any", "same", "few", "dropped", "none"])
@pytest.mark.parametrize("tokens,k,experts", [(1, 1, 1), (1, 8, 64), (63, 1, 5), (64, 1, 2), (65, 3, 7), (255, 2, 16), (257, 5, 128),
                                              (2048, 2, 64), (4096, 1, 1023), (4097, 1, 8), (1000, 8, 256), (1001, 4, 1024),
                                              (30, 2, 4000), (5000, 8, 4000), (70001, 1, 3), (65536, 8, 60)])
def test_order(tokens, k, experts, kind):
    ids = numbers(tokens, k, experts, tokens, kind)
    got = sort(ids, experts)
    for g, w, name in zip(got, plan(ids, experts), ("order", "slots", "offsets")):
        assert g.dtype == torch.int64 and np.array_equal(g.cpu().numpy(), w), name


def test_order_of_extreme_numbers():
    ids = np.array([[0, 2 ** 62, -2 ** 63], [2 ** 63 - 1, 2, 1], [2 ** 32, -1, 2 ** 32 + 1]])
    for g, w in zip(sort(ids, 3), plan(ids, 3)):
        assert np.array_equal(g.cpu().numpy(), w)


@pytest.mark.parametrize("tokens,k", [(0, 2), (5, 0), (0, 0)])
def test_no_assignments(tokens, k):
    from mask_loss_amd.functions import ExpertOrder, from_experts, to_experts
    order = sort(np.zeros((tokens, k), dtype=np.int64), 4)
    assert isinstance(order, ExpertOrder) and not order.offsets.any() and order.offsets.shape == (5,)
    x = torch.randn(tokens, 24, device="cuda", requires_grad=True)
    rows = to_experts(x, order)
    assert rows.shape == (0, 24)
    w = torch.ones(tokens, k, device="cuda", requires_grad=True)
    out = from_experts(rows, order, w)
    assert out.shape == (tokens, 24) and not out.any()
    gx, gw = torch.autograd.grad(out, (x, w), torch.ones_like(out))
    assert gx.shape == x.shape and not gx.any() and gw.shape == w.shape


def make(tokens, k, experts, D, dt, kind="dropped", params=None, seed=1):
    gen = torch.Generator().manual_seed(seed)
    ids = numbers(tokens, k, experts, seed, kind)
    t = TDT[dt]
    x, dout = (torch.randn(tokens, D, generator=gen).to(t) for _ in range(2))
    y, dxs = (torch.randn(tokens * k, D, generator=gen).to(t) for _ in range(2))
    w = torch.rand(tokens, k, generator=gen).to(TDT[params or dt])
    return ids, x, y, w, dxs, dout


def check(got, want, bound, name):
    assert got.shape == want.shape, name
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    err = (got.double().cpu() - want).abs()
    tol = bound + STEP[got.dtype] * want.abs() * (1 + 2 ** -7) + tiny + 1e-37
    assert not bool((~(err <= tol)).any()), (name, float((err / tol).max()))


def compare(ids, experts, x, y, w, dxs, dout, junk=True):
    from mask_loss_amd.functions import from_experts, to_experts
    T, k = ids.shape
    D = x.shape[1]
    order, slots, offsets = (torch.from_numpy(a) for a in plan(ids, experts))
    kept = int(offsets[-1])
    dev = sort(ids, experts)
    if junk:  # what lies in dropped places counts for nothing
        y, dxs = y.clone(), dxs.clone()
        y[kept:], dxs[kept:] = float("nan"), float("inf")
    leaves = [None if t is None else t.cuda().requires_grad_(True) for t in (x, y, w)]
    rows = to_experts(leaves[0], dev)
    want = torch.zeros(T * k, D, dtype=x.dtype)
    want[:kept] = x[order[:kept] // k]
    assert torch.equal(rows.detach().cpu(), want)
    out = from_experts(leaves[1], dev, leaves[2])
    given = [t for t in leaves if t is not None]
    grads = torch.autograd.grad((rows, out), given, (dxs.cuda(), dout.cuda()))

    at = order[:kept]
    wd = torch.ones(T * k, dtype=torch.float64) if w is None else w.double().reshape(-1)
    wy = y[:kept].double() * wd[at, None]
    zero = torch.zeros(T, D, dtype=torch.float64)
    check(out.detach(), zero.index_add(0, at // k, wy), (k + 1) * U * zero.index_add(0, at // k, wy.abs()), "out")
    dx = dxs[:kept].double()
    check(grads[0], zero.index_add(0, at // k, dx), (k + 1) * U * zero.index_add(0, at // k, dx.abs()), "dx")
    g = dout.double()[at // k]
    dy = torch.zeros(T * k, D, dtype=torch.float64)
    dy[:kept] = g * wd[at, None]
    check(grads[1], dy, U * dy.abs(), "drows")
    if w is None:
        return
    dw, bound = torch.zeros(T * k, dtype=torch.float64), torch.zeros(T * k, dtype=torch.float64)
    dw[at] = (g * y[:kept].double()).sum(1)
    bound[at] = (D / 16 + 8) * U * (g * y[:kept].double()).abs().sum(1)
    check(grads[2], dw.view(T, k), bound.view(T, k), "dw")
    assert grads[2].dtype == w.dtype


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [1, 2, 3, 8, 31, 32, 64, 100, 127, 128, 136, 256, 257, 512, 1000, 1024, 1153, 4096, 10000])
def test_widths(dt, D):
    compare(*(lambda a: (a[0], 6, *a[1:]))(make(23, 3, 6, D, dt)))


@pytest.mark.parametrize("params", ["f32", "bf16", None])
@pytest.mark.parametrize("tokens,k,experts,D,kind", [(1, 1, 1, 64, "any"), (1, 8, 16, 2048, "any"), (7, 1, 3, 40, "none"),
                                                     (2, 9, 4, 72, "dropped"), (3, 70, 20, 48, "dropped"), (3000, 2, 8, 64, "few"),
                                                     (40000, 1, 4, 33, "dropped"), (513, 8, 64, 256, "same")])
def test_sizes(tokens, k, experts, D, kind, params):
    args = make(tokens, k, experts, D, "bf16", kind, params or "bf16")
    if params is None:
        args = (*args[:3], None, *args[4:])
    compare(args[0], experts, *args[1:])


@pytest.mark.parametrize("dtype", [torch.uint8, torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.int64, torch.float64, torch.bool,
                                   torch.complex64])
@pytest.mark.parametrize("D", [1, 2, 6, 12, 17, 64, 1000])
def test_rows_of_any_type(dtype, D):
    from mask_loss_amd.functions import to_experts
    ids = numbers(50, 2, 5, 3, "dropped")
    order, _, offsets = plan(ids, 5)
    raw = torch.randint(0, 2 if dtype == torch.bool else 120, (50, D * torch.empty(0, dtype=dtype).element_size()),
                        generator=torch.Generator().manual_seed(4), dtype=torch.uint8)
    got = to_experts(raw.cuda().view(dtype), sort(ids, 5))
    want = torch.zeros(100, raw.shape[1], dtype=torch.uint8)
    want[:offsets[-1]] = raw[torch.from_numpy(order[:offsets[-1]] // 2)]
    assert got.dtype == dtype and torch.equal(got.view(torch.uint8).cpu(), want)


def test_layouts():
    """Transposed numbers, weights and rows, rows on no 16-byte boundary, upstream gradients that are broadcast."""
    from mask_loss_amd.functions import from_experts, sort_by_expert, to_experts
    ids, x, y, w, _, _ = make(40, 2, 6, 64, "bf16", "any")
    order = sort(ids, 6)
    turned = torch.from_numpy(np.ascontiguousarray(ids.T)).cuda().t()
    assert all(torch.equal(a, b) for a, b in zip(sort_by_expert(turned, 6), order))
    room = torch.empty(80 * 64 + 1, dtype=torch.bfloat16, device="cuda")
    for fn, t in ((lambda r: to_experts(r, order), x), (lambda r: from_experts(r, order, w.cuda()), y),
                  (lambda r: from_experts(r, order, w.cuda().t().contiguous().t()), y)):
        want = fn(t.cuda())
        leaf = t.cuda().requires_grad_(True)
        g, = torch.autograd.grad(fn(leaf), leaf, torch.ones_like(want))
        off = room[1:1 + t.numel()].view(t.shape).copy_(t)
        assert off.data_ptr() % 16 != 0
        for other in (off, t.cuda().t().contiguous().t(), torch.cat([t, t], 1).cuda()[:, :64]):
            assert torch.equal(fn(other), want)
            leaf = other.detach().requires_grad_(True)
            assert torch.equal(torch.autograd.grad(fn(leaf).sum(), leaf)[0], g)


def test_places_outside():
    """Places that point outside count as dropped: nothing is read or written there."""
    from mask_loss_amd.functions import ExpertOrder, from_experts, to_experts
    x, y = torch.randn(3, 32, device="cuda"), torch.randn(6, 32, device="cuda")
    slots = torch.tensor([[0, 6], [-1, 2 ** 62], [1, -2 ** 63]], device="cuda")
    for end, kept in ((6, 6), (2 ** 62, 6), (-5, 0), (1, 1)):
        offsets = torch.tensor([0, end], device="cuda")
        order = ExpertOrder(slots.flatten(), slots, offsets)
        room = torch.full((10, 32), 7.0, device="cuda")
        rows = to_experts(x, order)
        if kept > 0:
            assert torch.equal(rows[0], x[0])
        assert not rows[kept:].any()
        out = from_experts(y, order)
        assert torch.equal(out[0], y[0] if kept > 0 else torch.zeros_like(y[0])) and not out[1].any()
        assert torch.equal(out[2], y[1] if kept > 1 else torch.zeros_like(y[0]))
        leaf, w = y.clone().requires_grad_(True), torch.ones(3, 2, device="cuda", requires_grad=True)
        _, gw = torch.autograd.grad(from_experts(leaf, order, w), (leaf, w), torch.ones(3, 32, device="cuda"))
        assert not gw[1].any() and gw[0, 1] == 0 and gw[2, 1] == 0
        assert bool((room == 7.0).all())


def test_rows_past_32_bits():
    """4.3e9 elements there and back: each token's row twice, halved."""
    from mask_loss_amd.functions import from_experts, to_experts
    T, D = 1 << 21, 1040
    gen = torch.Generator(device="cuda").manual_seed(5)
    ids = torch.randint(0, 9, (T, 2), generator=gen, device="cuda")
    from mask_loss_amd.functions import sort_by_expert
    order = sort_by_expert(ids, 9)
    x = torch.randn(T, D, generator=gen, device="cuda").bfloat16()
    rows = to_experts(x, order)
    assert rows.numel() > 1 << 32
    at = order.order[-1000:]
    assert torch.equal(rows[-1000:], x[at // 2])
    w = torch.full((T, 2), 0.5, device="cuda")
    assert torch.equal(from_experts(rows, order, w), x)


def test_refusals():
    from mask_loss_amd.functions import ExpertOrder, from_experts, sort_by_expert, to_experts
    ids = torch.zeros(4, 2, dtype=torch.int64, device="cuda")
    for bad, E, words in ((ids.int(), 3, "int64"), (ids.flatten(), 3, "tokens, k"), (ids.cpu(), 3, "CUDA tensor"),
                          (ids, 0, "at least one expert"), (ids, 4001, "at most 4000")):
        with pytest.raises(RuntimeError, match=words):
            sort_by_expert(bad, E)
    order = sort_by_expert(ids, 3)
    x, y, w = torch.zeros(4, 8, device="cuda"), torch.zeros(8, 8, device="cuda"), torch.zeros(4, 2, device="cuda")
    for grad in (False, True):
        for bad, words in ((y, "with 4 rows"), (x[0], "with 4 rows"), (x.cpu(), "CUDA tensor")):
            with pytest.raises(RuntimeError, match=words):
                to_experts(bad.detach().requires_grad_(grad), order)
        for bad, wt, words in ((x, w, "with 8 rows"), (y.cpu(), w, "CUDA tensor"), (y, w[:3], "weights must be"),
                               (y, w.half(), "input's dtype"), (y.double(), None, "float32, bfloat16 or float16"),
                               (y, w.cpu(), "CUDA tensor")):
            with pytest.raises(RuntimeError, match=words):
                from_experts(bad.detach().requires_grad_(grad), order, wt)
        for bad in (ExpertOrder(order.order, order.slots.int(), order.offsets),
                    ExpertOrder(order.order, order.slots, order.offsets[:1]),
                    ExpertOrder(order.order, order.slots.cpu(), order.offsets)):
            with pytest.raises(RuntimeError, match="int64|offsets|CUDA tensor"):
                to_experts(x.detach().requires_grad_(grad), bad)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        to_experts(x.double().requires_grad_(True), order)
