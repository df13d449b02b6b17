"""CPU checks of calls that the head's operators (layer norm, grouped products, mask logits) refuse or answer
without the GPU, beside those of test_head_boundary.py, and of point sampling's forward mode."""
import pytest

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_params_f32_needs_a_float32_weight(dtype):
    """A 16-bit weight would be read as float32, past its end."""
    import mask_loss_amd
    x, stat = torch.zeros(4, 8, dtype=dtype), torch.zeros(4)
    with pytest.raises(RuntimeError, match="float32 weight"):
        mask_loss_amd.mask_loss.layer_norm_backward(x, x, torch.ones(8, dtype=dtype), stat, stat, params_f32=True)


def test_tangents_are_refused():
    """A tensor that carries a tangent: every form raises, none leaves the tangent behind."""
    import mask_loss_amd
    from torch.autograd import forward_ad
    from mask_loss_amd.functions import grouped_matmul, layer_norm, mask_logits
    ml = mask_loss_amd.mask_loss
    x, w, b, wg = torch.ones(4, 8), torch.ones(8), torch.zeros(8), torch.zeros(2, 8, 3)
    o, stat, q, f = torch.tensor([0, 2, 4]), torch.zeros(4), torch.zeros(1, 2, 3, 8), torch.zeros(2, 8, 5, 5)
    calls = [(layer_norm, (x, w, b), 3), (grouped_matmul, (x, wg, o), 2), (mask_logits, (q, f), 2),
             (mask_logits, (x, f, o), 2), (ml.layer_norm_backward, (x, x, w, stat, stat), 5),
             (ml.grouped_matmul_backward_input, (torch.ones(4, 3), wg, o), 2),
             (ml.grouped_matmul_backward_weight, (x, torch.ones(4, 3), o, 2), 2)]
    with forward_ad.dual_level():
        for fn, args, n in calls:
            for i in range(n):
                for grad in (False, True):
                    these = [t.clone() if torch.is_tensor(t) else t for t in args]
                    these[i] = forward_ad.make_dual(these[i], torch.ones_like(these[i]))
                    if grad:
                        these[0].requires_grad_(True)
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        fn(*these)


def test_point_sample_refuses_tangents():
    import mask_loss_amd
    from torch.autograd import forward_ad
    from mask_loss_amd.functions import point_sample
    x, c, g = torch.ones(2, 3, 4, 4), torch.zeros(2, 5, 2), torch.ones(2, 3, 5)
    with forward_ad.dual_level():
        for fn, args in ((point_sample, (x, c)), (mask_loss_amd.mask_loss.point_sample_backward, (g, c, 4, 4, False))):
            for i in (0, 1):
                these = list(args)
                these[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    fn(*these)
