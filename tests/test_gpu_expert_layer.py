"""The operators around the head's grouped products as a program uses them: an expert layer with its residual in training and
in inference, captured steps, other streams, two threads, and the calls that the tests of one operator each do not make."""
import threading

import pytest

torch = pytest.importorskip("torch")

import mx_reference as mx  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


E, K, D, H = 6, 2, 96, 160


def layer(x, residual, wn, ids, gates, w1, w2):
    """norm of the sum, rows to their experts, two products, back with the gates, and the norm behind"""
    from mask_loss_amd.functions import from_experts, grouped_matmul, rms_norm, sort_by_expert, to_experts
    h, s = rms_norm(x, wn, 1e-6, residual)
    order = sort_by_expert(ids, w1.shape[0])
    rows = to_experts(h, order)
    rows = grouped_matmul(rows, w1, order.offsets, transposed=True)
    rows = grouped_matmul(rows * torch.sigmoid(rows), w2, order.offsets, transposed=True)
    return rms_norm(from_experts(rows, order, gates), wn, 1e-6, s)


def plain_layer(x, residual, wn, ids, gates, w1, w2):
    def norm(t):
        return t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * wn
    s = x + residual
    h = norm(s)
    out = torch.zeros_like(h)
    for j in range(ids.shape[1]):
        for e in range(w1.shape[0]):
            pick = (ids[:, j] == e).to(h.dtype)[:, None]
            r = h @ w1[e].t()
            out = out + pick * gates[:, j:j + 1] * ((r * torch.sigmoid(r)) @ w2[e].t())
    return norm(out + s), out + s


def make(tokens, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x, res, dy, ds = (torch.randn(tokens, D, generator=gen) for _ in range(4))
    wn = 1 + 0.2 * torch.randn(D, generator=gen)
    ids = torch.randint(-1, E + 1, (tokens, K), generator=gen)
    gates = torch.rand(tokens, K, generator=gen)
    w1, w2 = torch.randn(E, H, D, generator=gen) * D ** -0.5, torch.randn(E, D, H, generator=gen) * H ** -0.5
    return [t.to(dtype) if t.is_floating_point() else t for t in (x, res, wn, ids, gates, w1, w2)], dy.to(dtype), ds.to(dtype)


@pytest.mark.parametrize("tokens", [1, 7, 300])
def test_layer_trains(tokens):
    """float32 against the definition in float64: outputs and all gradients, in the large (2e-5 of each one's size: about
    D + H + D additions of 2^-24 each in a row, which grow at most a few times over on their way)."""
    args, dy, ds = make(tokens, torch.float32, tokens)
    leaves = [t.cuda().requires_grad_(True) if t.is_floating_point() else t.cuda() for t in args]
    outs = layer(*leaves)
    wanted = [t for t in leaves if t.requires_grad]
    grads = torch.autograd.grad(outs, wanted, (dy.cuda(), ds.cuda()))
    exact = [t.double().requires_grad_(True) if t.is_floating_point() else t for t in args]
    ref = plain_layer(*exact)
    want = torch.autograd.grad(ref, [t for t in exact if t.requires_grad], (dy.double(), ds.double()))
    for got, w in zip((*outs, *grads), (*ref, *want)):
        assert float((got.detach().double().cpu() - w.detach()).norm()) <= 2e-5 * float(w.detach().norm()) + 1e-12


def test_layer_trains_in_16_bits():
    """bfloat16 against float64: every tensor between two operators is rounded by 2^-8 at most, seven in a row, and their
    errors add up in the mean (4 steps) rather than in the worst case."""
    args, dy, ds = make(200, torch.bfloat16, 5)
    leaves = [t.cuda().requires_grad_(True) if t.is_floating_point() else t.cuda() for t in args]
    outs = layer(*leaves)
    grads = torch.autograd.grad(outs, [t for t in leaves if t.requires_grad], (dy.cuda(), ds.cuda()))
    exact = [t.double().requires_grad_(True) if t.is_floating_point() else t for t in args]
    ref = plain_layer(*exact)
    want = torch.autograd.grad(ref, [t for t in exact if t.requires_grad], (dy.double(), ds.double()))
    for got, w in zip((*outs, *grads), (*ref, *want)):
        assert got.dtype == torch.bfloat16
        assert float((got.detach().double().cpu() - w.detach()).norm()) <= 4 * 2.0 ** -8 * float(w.detach().norm())


def serve(x, residual, wn, ids, gates, w1, w2):
    """The same with quantised operands; w1, w2: (codes, scales)"""
    from mask_loss_amd.functions import (from_experts, grouped_matmul_mx, mx_quantize, rms_norm, rms_norm_mx, sort_by_expert,
                                         to_experts)
    codes, scales, s = rms_norm_mx(x, wn, 1e-6, residual)
    order = sort_by_expert(ids, w1[0].shape[0])
    rows = grouped_matmul_mx(to_experts(codes, order), to_experts(scales, order), *w1, order.offsets, dtype=x.dtype)
    rows = grouped_matmul_mx(*mx_quantize(rows * torch.sigmoid(rows)), *w2, order.offsets, dtype=x.dtype)
    return rms_norm(from_experts(rows, order, gates), wn, 1e-6, s)


def quantised(w, format):
    from mask_loss_amd.functions import mx_quantize
    return mx_quantize(w.cuda(), format)


@pytest.mark.parametrize("format", ["e2m1", "e4m3"])
@pytest.mark.parametrize("tokens", [1, 16, 500])
def test_layer_serves(tokens, format):
    """Step by step what its operators give, and near the layer of the dequantised weights: activations in e4m3 are off by
    2^-4 of their value each at most, 2^-5 in the mean of squares, over two products and a norm."""
    args, _, _ = make(tokens, torch.bfloat16, tokens + 1)
    x, res, wn, ids, gates = (t.cuda() for t in args[:5])
    w1, w2 = quantised(args[5], format), quantised(args[6], format)
    y, s = serve(x, res, wn, ids, gates, w1, w2)
    exact = [t.double() if t.is_floating_point() else t for t in args[:5]]
    ref = plain_layer(*exact, mx.decode(*w1), mx.decode(*w2))
    for got, w in zip((y, s), ref):
        assert float((got.double().cpu() - w).norm()) <= 2 * 2.0 ** -5 * float(w.norm())


def test_captured_layers():
    """Training and serving steps captured into two graphs, replayed in turn with other inputs, experts and gates, eager
    work between: each replay as the eager call."""
    args, dy, ds = make(120, torch.bfloat16, 3)
    leaves = [t.cuda().requires_grad_(True) if t.is_floating_point() else t.cuda() for t in args]
    dyd, dsd = dy.cuda(), ds.cuda()
    wanted = [t for t in leaves if t.requires_grad]
    w1, w2 = quantised(args[5], "e2m1"), quantised(args[6], "e4m3")

    def train():
        outs = layer(*leaves)
        return (*[t.detach() for t in outs], *torch.autograd.grad(outs, wanted, (dyd, dsd)))

    def infer():
        with torch.no_grad():
            return serve(*leaves[:5], w1, w2)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train()
        infer()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for step in (train, infer):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs, step))
    for seed in (11, 12, 13):
        new, dy, ds = make(120, torch.bfloat16, seed)
        with torch.no_grad():
            for t, n in zip(leaves, new):
                t.copy_(n)
            dyd.copy_(dy)
            dsd.copy_(ds)
        for graph, outs, step in graphs:
            for t in outs:
                t.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, step()))


def test_sorts_captured_in_one_and_several_workgroups():
    from mask_loss_amd.functions import sort_by_expert
    for tokens in (500, 9000):
        ids = torch.randint(0, 40, (tokens, 3), device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = sort_by_expert(ids, 33)
        for seed in range(3):
            ids.copy_(torch.randint(0, 40, (tokens, 3), generator=torch.Generator().manual_seed(seed)))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, sort_by_expert(ids, 33)))


def operator(name):
    """(call, leaves, upstream gradient) of a small training call"""
    from mask_loss_amd.functions import from_experts, rms_norm, sort_by_expert, to_experts
    gen = torch.Generator().manual_seed(3)

    def leaf(*shape):
        return torch.randn(*shape, generator=gen).bfloat16().cuda().requires_grad_(True)

    order = sort_by_expert(torch.randint(0, 5, (40, 2), generator=gen).cuda(), 4)
    torch.cuda.synchronize()
    if name == "rms_norm":
        return (lambda x, w, r: rms_norm(x, w, 1e-6, r)[0]), [leaf(40, 64), leaf(64), leaf(40, 64)], leaf(40, 64).detach()
    if name == "rms_norm_sum":
        return (lambda x, w, r: rms_norm(x, w, 1e-6, r)[1]), [leaf(40, 64), leaf(64), leaf(40, 64)], leaf(40, 64).detach()
    if name == "to_experts":
        return (lambda x: to_experts(x, order)), [leaf(40, 64)], leaf(80, 64).detach()
    return (lambda y, w: from_experts(y, order, w)), [leaf(80, 64), leaf(40, 2)], leaf(40, 64).detach()


NAMES = ["rms_norm", "rms_norm_sum", "to_experts", "from_experts"]


def grads_of(y, leaves, dy, **kw):
    return [g for g in torch.autograd.grad(y, leaves, dy, allow_unused=True, **kw) if g is not None]


@pytest.mark.parametrize("name", NAMES)
def test_captured_backward_beside_an_eager_graph(name):
    """While an eager call's output is alive its leaves' gradients belong to the default stream: a captured
    backward into one of them is refused, the captured forward is not, and both work when it is gone."""
    fn, leaves, dy = operator(name)
    want = fn(*leaves)
    want_grads = grads_of(want, leaves, dy, retain_graph=True)
    torch.cuda.synchronize()
    for i in range(len(leaves)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = fn(*leaves)
            with pytest.raises(RuntimeError, match="cannot be captured"):
                torch.autograd.grad(y, leaves[i], dy)
        for _ in range(2):
            y.detach().zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want)
        del y, graph
    value = want.detach().clone()
    del want  # the eager graph and its nodes
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fn(*leaves)
        grads = grads_of(y, leaves, dy)
    for _ in range(3):
        for t in (y.detach(), *(g for g in grads if g.data_ptr() != dy.data_ptr())):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, value) and all(torch.equal(a, b) for a, b in zip(grads, want_grads))


@pytest.mark.parametrize("name", NAMES)
def test_two_threads_at_once(name):
    """Training calls of two host threads on streams of their own, side by side: each as alone."""
    fn, leaves, dy = operator(name)
    want = fn(*leaves).detach()
    want_grads = grads_of(fn(*leaves), leaves, dy)
    torch.cuda.synchronize()
    start, bad = threading.Barrier(2), []

    def work():
        own = [t.detach().clone().requires_grad_(True) for t in leaves]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        start.wait(30)
        with torch.cuda.stream(stream):
            outs = []
            for _ in range(20):
                y = fn(*own)
                outs.append((y.detach(), grads_of(y, own, dy)))
        stream.synchronize()
        for y, grads in outs:
            if not torch.equal(y, want) or not all(torch.equal(a, b) for a, b in zip(grads, want_grads)):
                bad.append(name)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not any(t.is_alive() for t in threads) and not bad


def test_serving_on_other_streams_and_threads():
    """The serving layer on two streams by two threads: workspaces of split products are each call's own."""
    from mask_loss_amd.functions import grouped_matmul_mx
    args, _, _ = make(64, torch.bfloat16, 9)
    x, res, wn, ids, gates = (t.cuda() for t in args[:5])
    w1, w2 = quantised(args[5], "e2m1"), quantised(args[6], "e2m1")
    long = quantised(torch.randn(200, 8192).bfloat16(), "e4m3"), quantised(torch.randn(1, 96, 8192).bfloat16(), "e2m1")
    o = torch.tensor([0, 200], device="cuda")
    want = (*serve(x, res, wn, ids, gates, w1, w2), grouped_matmul_mx(*long[0], *long[1], o))
    torch.cuda.synchronize()
    bad, start = [], threading.Barrier(2)

    def work():
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.default_stream())
        start.wait(30)
        with torch.cuda.stream(stream), torch.no_grad():
            outs = [(*serve(x, res, wn, ids, gates, w1, w2), grouped_matmul_mx(*long[0], *long[1], o)) for _ in range(20)]
        stream.synchronize()
        if not all(torch.equal(a, b) for out in outs for a, b in zip(out, want)):
            bad.append(1)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not any(t.is_alive() for t in threads) and not bad


@pytest.mark.parametrize("name", NAMES)
def test_inference_mode_and_equal_runs(name):
    fn, leaves, dy = operator(name)
    want = fn(*leaves).detach()
    with torch.inference_mode():
        assert torch.equal(fn(*[t.clone() for t in leaves]), want)
        assert torch.equal(fn(*leaves), want)
    first = grads_of(fn(*leaves), leaves, dy)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(grads_of(fn(*leaves), leaves, dy), first))


@pytest.mark.parametrize("name", NAMES)
def test_second_derivative_is_refused(name):
    fn, leaves, dy = operator(name)
    y = fn(*leaves)
    g, = torch.autograd.grad(y.square().sum(), leaves[0], create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        g.sum().backward()


@pytest.mark.parametrize("name", NAMES)
def test_upstream_gradients_with_tangents_are_refused(name):
    from torch.autograd import forward_ad
    fn, leaves, dy = operator(name)
    with forward_ad.dual_level():
        y = fn(*leaves)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, leaves[0], forward_ad.make_dual(dy, torch.ones_like(dy)))


def test_gradients_against_differences():
    """Rows there and back: the gradients along random directions against central differences of the float64 definition
    (which is linear in each argument: no error of the differences)."""
    from mask_loss_amd.functions import from_experts, sort_by_expert, to_experts
    gen = torch.Generator().manual_seed(6)
    ids = torch.randint(-1, 6, (30, 3), generator=gen)
    x, up, g = torch.randn(30, 40, generator=gen), torch.randn(30, 40, generator=gen), torch.rand(30, 3, generator=gen)
    scale = torch.randn(90, 1, generator=gen)
    order = sort_by_expert(ids.cuda(), 5)
    leaves = [t.cuda().requires_grad_(True) for t in (x, g)]
    out = from_experts(to_experts(leaves[0], order) * scale.cuda(), order, leaves[1])
    grads = torch.autograd.grad(out, leaves, up.cuda())
    slots, kept = order.slots.cpu(), int(order.offsets[-1])

    def loss(x, g):
        w = torch.where(slots < kept, g * scale.double()[slots, 0], 0.0).sum(1, keepdim=True)
        return float((w * x * up.double()).sum())

    args = [x.double(), g.double()]
    for i, grad in enumerate(grads):
        v = torch.randn(args[i].shape, generator=gen, dtype=torch.float64)
        hi, lo = ([t + k * v if j == i else t for j, t in enumerate(args)] for k in (1, -1))
        want = (loss(*hi) - loss(*lo)) / 2
        # float32 sums of 40 and 3 terms
        assert abs(float((grad.double().cpu() * v).sum()) - want) <= 64 * 2.0 ** -24 * float((grad.double().cpu() * v).abs().sum())


def test_views():
    """Views that share memory, and weights that are one value for all (a broadcast view): each as its copy."""
    from mask_loss_amd.functions import from_experts, rms_norm, sort_by_expert, to_experts
    base = torch.randn(41, 64, device="cuda").bfloat16()
    a, b = base[:40], base[1:]
    w = torch.tensor([1.5], device="cuda").bfloat16().expand(64).requires_grad_(True)
    y, s = rms_norm(a, w, 1e-6, b)
    y2, s2 = rms_norm(a.clone(), w.detach().contiguous(), 1e-6, b.clone())
    assert torch.equal(y, y2) and torch.equal(s, s2)
    gw, = torch.autograd.grad(y, w, torch.ones_like(y))
    assert gw.shape == (64,)
    order = sort_by_expert(torch.randint(0, 4, (40, 2), device="cuda"), 4)
    one = torch.ones((), device="cuda").expand(40, 2).requires_grad_(True)
    rows = to_experts(a, order)
    out = from_experts(rows, order, one)
    assert torch.equal(out, from_experts(rows, order))
    g, = torch.autograd.grad(out, one, torch.ones_like(out))
    assert g.shape == (40, 2)


def memory(t):
    return t.untyped_storage().data_ptr()


@pytest.mark.parametrize("name", NAMES)
def test_gradients_have_their_own_memory(name):
    """Gradients that accumulate in leaves share memory with no upstream gradient and with no other leaf's: a second backward
    and zero_() change each leaf's alone."""
    fn, leaves, dy = operator(name)
    want = torch.autograd.grad(fn(*leaves), leaves, dy, allow_unused=True)
    want = [None if g is None else g.clone() for g in want]
    up = dy.clone()
    fn(*leaves).backward(up)
    given = [(t, g) for t, g in zip(leaves, want) if g is not None]
    assert len({memory(up), *[memory(t.grad) for t, _ in given]}) == len(given) + 1
    assert all(torch.equal(t.grad, g) for t, g in given)
    fn(*leaves).backward(up)
    assert torch.equal(up, dy) and all(torch.equal(t.grad, g + g) for t, g in given)
    given[0][0].grad.zero_()
    assert torch.equal(up, dy) and all(torch.equal(t.grad, g + g) for t, g in given[1:])


@pytest.mark.parametrize("residual_wanted", [False, True])
def test_the_sum_beside_another_user_of_its_gradient(residual_wanted):
    """The sum alone, added to another leaf, whose gradient is the sum's upstream one: accumulated twice, clipped in
    place, and in a broadcast form."""
    from mask_loss_amd.functions import rms_norm
    x, other = (torch.randn(40, 64, device="cuda").requires_grad_(True) for _ in range(2))
    res = torch.randn(40, 64, device="cuda").requires_grad_(residual_wanted)
    w = torch.ones(64, device="cuda", requires_grad=True)
    leaves = [t for t in (x, other, res) if t.requires_grad]
    for up in (torch.ones(40, 64, device="cuda"), torch.ones((), device="cuda").expand(40, 64)):
        ((rms_norm(x, w, 1e-6, res)[1] + other) * 1.0).backward(up)
    assert all(bool((t.grad == 2).all()) for t in leaves)
    assert len({memory(t.grad) for t in leaves}) == len(leaves)
    x.grad.clamp_(max=0.5)
    assert bool((x.grad == 0.5).all()) and all(bool((t.grad == 2).all()) for t in leaves[1:])
    assert w.grad is None or not w.grad.any()
    up = torch.full((40, 64), 3.0, device="cuda")
    g, = torch.autograd.grad(rms_norm(x, w, 1e-6, res)[1], x, up)
    assert memory(g) != memory(up) and bool((g == 3).all())


@pytest.mark.parametrize("grad", [True, False])
def test_function_classes(grad):
    """The operators' Function classes: results and gradients of the functions, with and without leaves that want them."""
    from mask_loss_amd.functions import (FromExpertsFunction, RMSNormFunction, ToExpertsFunction, from_experts, rms_norm,
                                         sort_by_expert, to_experts)
    gen = torch.Generator().manual_seed(8)
    x, res = (torch.randn(40, 64, generator=gen).cuda() for _ in range(2))
    w, y, g = torch.randn(64, generator=gen).cuda(), torch.randn(80, 64, generator=gen).cuda(), torch.rand(40, 2, generator=gen).cuda()
    order = sort_by_expert(torch.randint(-1, 5, (40, 2), generator=gen).cuda(), 4)
    calls = [(lambda a: RMSNormFunction.apply(a), rms_norm, (x,)),
             (lambda a, b: RMSNormFunction.apply(a, b, 1e-5), lambda a, b: rms_norm(a, b, 1e-5), (x, w)),
             (lambda a, b, c: RMSNormFunction.apply(a, b, 1e-5, c), lambda a, b, c: rms_norm(a, b, 1e-5, c), (x, w, res)),
             (lambda a: ToExpertsFunction.apply(a, order.slots, order.offsets), lambda a: to_experts(a, order), (x,)),
             (lambda a: FromExpertsFunction.apply(a, order.slots, order.offsets), lambda a: from_experts(a, order), (y,)),
             (lambda a, b: FromExpertsFunction.apply(a, order.slots, order.offsets, b), lambda a, b: from_experts(a, order, b), (y, g))]
    for one, other, args in calls:
        leaves = [t.clone().requires_grad_(grad) for t in args]
        got, want = ([o] if isinstance(o, torch.Tensor) else list(o) for o in (one(*leaves), other(*leaves)))
        assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(o.requires_grad == grad for o in got)
        if grad:
            ups = [torch.randn(o.shape, generator=gen).cuda() for o in got]
            assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, leaves, ups), torch.autograd.grad(want, leaves, ups)))
