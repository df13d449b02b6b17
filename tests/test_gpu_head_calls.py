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
