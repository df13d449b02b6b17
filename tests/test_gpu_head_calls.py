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
