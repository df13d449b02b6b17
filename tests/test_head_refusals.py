"""CPU checks of calls that the head's operators (layer norm, grouped products, mask logits) refuse or answer
without the GPU, beside those of test_head_boundary.py."""
import pytest

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_params_f32_needs_a_float32_weight(dtype):
    """A 16-bit weight would be read as float32, past its end."""
    import mask_loss_amd
    x, stat = torch.zeros(4, 8, dtype=dtype), torch.zeros(4)
    with pytest.raises(RuntimeError, match="float32 weight"):
        mask_loss_amd.mask_loss.layer_norm_backward(x, x, torch.ones(8, dtype=dtype), stat, stat, params_f32=True)
