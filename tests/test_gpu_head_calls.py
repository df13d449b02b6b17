"""Calls of the head's operators (layer norm, grouped products, mask logits) on the GPU that the tests
of one operator each do not make."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def test_upstream_gradients_with_tangents_are_refused():
    from torch.autograd import forward_ad
    from mask_loss_amd.functions import grouped_matmul, layer_norm, mask_logits
    x, w = torch.ones(4, 8, device="cuda"), torch.ones(2, 8, 3, device="cuda")
    q, f = torch.ones(1, 2, 4, 8, device="cuda"), torch.ones(2, 8, 5, 5, device="cuda")
    o = torch.tensor([0, 2, 4], device="cuda")
    for fn, args in ((layer_norm, (x,)), (grouped_matmul, (x, w, o)), (mask_logits, (q, f))):
        leaf = args[0].clone().requires_grad_(True)
        with forward_ad.dual_level():
            y = fn(leaf, *args[1:])
            dy = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(y, leaf, dy)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                fn(forward_ad.make_dual(args[0], args[0]), *args[1:])


@pytest.mark.parametrize("rows", [0, 5])
def test_mask_logits_of_no_image(rows):
    """A ragged set for an empty batch: rows in no image's set give zeros."""
    from mask_loss_amd.functions import mask_logits
    q = torch.randn(rows, 8, device="cuda", requires_grad=True)
    f = torch.zeros(0, 8, 4, 6, device="cuda", requires_grad=True)
    o = torch.zeros(1, dtype=torch.int64, device="cuda")
    z = mask_logits(q, f, o)
    assert z.shape == (rows, 4, 6) and not z.any()
    dq, df = torch.autograd.grad(z, (q, f), torch.ones_like(z))
    assert dq.shape == q.shape and not dq.any() and df.shape == f.shape
    with torch.no_grad():
        assert torch.equal(mask_logits(q, f, o), z)
        for bad, words in (((q, f, o.int()), "int64"), ((q, f.half(), o), "same dtype"), ((q, f, o.cpu()), "CUDA tensor")):
            with pytest.raises(RuntimeError, match=words):
                mask_logits(*bad)


def operator(name):
    """(call, leaves, upstream gradient) of a small training call"""
    from mask_loss_amd.functions import grouped_matmul, layer_norm, mask_logits
    gen = torch.Generator().manual_seed(3)

    def leaf(*shape):
        return torch.randn(*shape, generator=gen).bfloat16().cuda().requires_grad_(True)

    if name == "layer_norm":
        return layer_norm, [leaf(40, 64), leaf(64), leaf(64)], torch.ones(40, 64, device="cuda").bfloat16()
    if name == "mask_logits":
        return mask_logits, [leaf(2, 2, 5, 64), leaf(2, 64, 8, 8)], torch.ones(2, 2, 5, 8, 8, device="cuda").bfloat16()
    o = torch.tensor([0, 30, 40], device="cuda")
    return (lambda x, w: grouped_matmul(x, w, o)), [leaf(40, 64), leaf(2, 64, 72)], torch.ones(40, 72, device="cuda").bfloat16()


@pytest.mark.parametrize("name", ["layer_norm", "grouped_matmul", "mask_logits"])
def test_captured_backward_beside_an_eager_graph(name):
    """While an eager call's output is alive its leaves' gradients belong to the default stream: a captured
    backward into one of them is refused, the captured forward is not, and both work when it is gone."""
    fn, leaves, dy = operator(name)
    want = fn(*leaves)
    want_grads = torch.autograd.grad(want, leaves, dy, retain_graph=True)
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
        grads = torch.autograd.grad(y, leaves, dy)
    for _ in range(3):
        for t in (y.detach(), *grads):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, value) and all(torch.equal(a, b) for a, b in zip(grads, want_grads))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("K,N", [(1 << 22, 8), ((1 << 22) - 3, 5), (8, 1 << 22), (5, (1 << 22) - 3)])
def test_longest_reductions_and_rows(dt, K, N):
    """K and N up to 2^22, the most that the products take."""
    import test_gpu_grouped as grouped
    x, w, dy = grouped.make(7, K, N, 2, dt, False, 5)
    grouped.compare(x, w, dy, [1, 3, 6], False)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_widest_norm(dt):
    """A width of 2^26, the most that the norm takes: a thread adds width / 1024 terms."""
    import test_gpu_norm as norm
    D = 1 << 26
    gen = torch.Generator(device="cuda").manual_seed(8)
    x, dy = ((torch.randn(2, D, generator=gen, device="cuda") + s).to(norm.TDT[dt]) for s in (0.5, 0.0))
    w, b = ((1 + 0.2 * torch.randn(D, generator=gen, device="cuda")).to(norm.TDT[dt]) for _ in range(2))
    got = norm.run(x, w, b, dy)
    ref = norm.reference(x, w, b.double(), dy, 1e-5, 64 + D // 1024)
    for g, (v, bound), name in zip(got, ref, ("y", "dx", "dw", "db")):
        tol = bound + norm.STEP[g.dtype] * v.abs() * (1 + 2 ** -7) + 1e-37
        assert bool(((g.double() - v).abs() <= tol).all()), name


@pytest.mark.parametrize("name", ["layer_norm", "grouped_matmul", "mask_logits"])
def test_two_threads_at_once(name):
    """Training calls of two host threads on streams of their own, side by side: each as alone."""
    import threading
    fn, leaves, dy = operator(name)
    want = fn(*leaves).detach()
    want_grads = torch.autograd.grad(fn(*leaves), leaves, dy)
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
                outs.append((y.detach(), torch.autograd.grad(y, own, dy)))
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


@pytest.mark.parametrize("K,rows,offsets", [(64, 40, [0, 10, 40]), (61, 400, [0, 200, 400]), (64, 400, [0, 200, 400])])
@pytest.mark.parametrize("transposed", [False, True])
def test_small_float16_values(K, rows, offsets, transposed):
    """float16 inputs below the normal range (2^-14) count in full, and so do outputs there: each kernel."""
    import test_gpu_grouped as grouped
    x, w, dy = grouped.make(rows, K, 72, 2, "f16", transposed, 9)
    x, dy = (x.float() * 2.0 ** -16).half(), (dy.float() * 2.0 ** -13).half()
    assert bool((x.abs() < 2.0 ** -14).float().mean() > 0.9)
    grouped.compare(x, (w.float() * 64).half(), dy, offsets, transposed)
    grouped.compare(x, w, dy, offsets, transposed)


@pytest.mark.parametrize("name", ["layer_norm", "grouped_matmul", "mask_logits"])
def test_inference_mode(name):
    fn, leaves, _ = operator(name)
    want = fn(*leaves).detach()
    with torch.inference_mode():
        assert torch.equal(fn(*[t.clone() for t in leaves]), want)
        assert torch.equal(fn(*leaves), want)
