"""Microscaled values on the GPU: codes and scales equal to the float64 definition's, bit by bit."""
import pytest

torch = pytest.importorskip("torch")

import mx_reference as mx  # noqa: E402

pytestmark = pytest.mark.gpu

TDT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module", autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def check(x, format):
    from mask_loss_amd.functions import mx_quantize
    codes, scales = mx_quantize(x.cuda(), format)
    assert scales.dtype == torch.float8_e8m0fnu and scales.shape == (*x.shape[:-1], x.shape[-1] // 32)
    assert codes.dtype == (torch.uint8 if format == "e2m1" else torch.float8_e4m3fn)
    assert codes.shape == (*x.shape[:-1], x.shape[-1] // (2 if format == "e2m1" else 1))
    q, b = mx.quantize(x, format)
    assert torch.equal(mx.byte(scales), b)
    assert torch.equal(mx.values(codes), q)
    assert torch.equal(torch.signbit(mx.values(codes)), torch.signbit(q))


@pytest.mark.parametrize("format", ["e2m1", "e4m3"])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(1, 32), (32,), (7, 64), (2, 3, 96), (1001, 160), (5, 8192), (40000, 32), (0, 64), (3, 0)])
def test_shapes(format, dt, shape):
    gen = torch.Generator().manual_seed(len(shape))
    check((torch.randn(shape, generator=gen) * torch.exp(3 * torch.randn(shape, generator=gen))).to(TDT[dt]), format)


@pytest.mark.parametrize("format", ["e2m1", "e4m3"])
def test_values(format):
    """Every value of the format and every midpoint between two, and their neighbours, beside a largest one of each
    kind; blocks of zeros; the smallest and largest floats; NaN and infinities."""
    every = mx.E2M1 if format == "e2m1" else torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = torch.cat([every, (every[1:] + every[:-1]) / 2]).float()
    near = torch.cat([mid, torch.nextafter(mid, torch.tensor(1e9)), torch.nextafter(mid, torch.tensor(-1e9))])
    near = torch.cat([near, -near])
    near = torch.cat([near, near.new_zeros(-near.numel() % 31)]).view(-1, 31)
    top = 2.0 ** mx.EMAX[format]
    for largest in (top, top * 1.25, top * 1.75, top * 1.96875, top * (2 - 2.0 ** -23)):
        block = torch.cat([torch.full((near.shape[0], 1), largest), near.clamp(-largest, largest)], 1)
        for e in (0, 1, -20, 100, -110):
            check(block * 2.0 ** e, format)
    gen = torch.Generator().manual_seed(2)
    wild = torch.randint(-2 ** 31, 2 ** 31, (500, 32), generator=gen).int().view(torch.float32)  # any bits
    check(wild, format)
    for x in (torch.zeros(2, 32), -torch.zeros(2, 32), torch.full((1, 32), 3.4028234e38), torch.full((1, 32), 2.0 ** -149),
              torch.full((1, 32), 2.0 ** -126), torch.arange(32).float().view(1, 32) * 2.0 ** -149,
              torch.arange(32).float().view(1, 32) * 2.0 ** -130):
        check(x, format)
    for bad in (float("nan"), float("inf"), float("-inf")):
        x = torch.randn(4, 96, generator=gen)
        x[1, 40], x[2, 95], x[3, 0] = bad, bad, bad
        check(x, format)
        check(x.bfloat16(), format)


def test_layouts():
    from mask_loss_amd.functions import mx_quantize
    x = torch.randn(64, 96).bfloat16()
    want = mx_quantize(x.cuda(), "e2m1")
    room = torch.empty(64 * 96 + 1, dtype=torch.bfloat16, device="cuda")
    off = room[1:].view(64, 96).copy_(x)
    assert off.data_ptr() % 16 != 0
    for other in (off, x.cuda().t().contiguous().t(), torch.cat([x, x], 1).cuda()[:, :96]):
        got = mx_quantize(other, "e2m1")
        assert torch.equal(got[0], want[0]) and torch.equal(mx.byte(got[1]), mx.byte(want[1]))


def test_past_32_bits():
    from mask_loss_amd.functions import mx_quantize
    x = torch.zeros(1 << 22, 1056, dtype=torch.bfloat16, device="cuda")
    x[-5:] = torch.randn(5, 1056, device="cuda").bfloat16()
    codes, scales = mx_quantize(x)
    c, s = mx_quantize(x[-5:])
    assert torch.equal(codes[-5:].view(torch.uint8), c.view(torch.uint8)) and torch.equal(mx.byte(scales[-5:]), mx.byte(s))


def test_refusals():
    from mask_loss_amd.functions import mx_quantize
    x = torch.zeros(4, 64, device="cuda")
    for bad, words in ((x[:, :48], "multiple of 32"), (x.double(), "float32, bfloat16 or float16"), (x.cpu(), "CUDA tensor"),
                       (x[0, 0], "multiple of 32")):
        with pytest.raises(RuntimeError, match=words):
            mx_quantize(bad)
    with pytest.raises(ValueError, match="format"):
        mx_quantize(x, "e5m2")
    with pytest.raises(NotImplementedError, match="no gradient"):
        mx_quantize(x.requires_grad_(True))
