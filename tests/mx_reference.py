"""Microscaled values in float64 on the CPU, for the tests."""
import torch

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
LARGEST = {"e2m1": 6.0, "e4m3": 448.0}
EMAX = {"e2m1": 2, "e4m3": 8}
FRACTION = {"e2m1": 1, "e4m3": 3}
EMIN = {"e2m1": 0, "e4m3": -6}


def nearest(q, format):
    """The format's value nearest to each of q, ties to the even fraction, held to the largest."""
    m = q.abs()
    e = torch.frexp(m).exponent - 1
    step = torch.exp2((torch.where(m > 0, e, EMIN[format]).clamp_min(EMIN[format]) - FRACTION[format]).double())
    return torch.copysign((torch.round(m / step) * step).clamp_max(LARGEST[format]), q)


def scale_codes(x, format):
    """int64 codes of the scales of x's blocks of 32: exponent and 127, 255 for NaN."""
    top = x.double().unflatten(-1, (-1, 32)).abs().amax(-1)
    e = (torch.frexp(top).exponent - 1 - EMAX[format]).clamp(-127, 127)
    e = torch.where(top > 0, e, -127)
    return torch.where(torch.isfinite(top), e + 127, 255)


def divide(x, codes):
    """x / scale, zeros in the blocks whose scale is NaN"""
    v = x.double().unflatten(-1, (-1, 32)) / torch.exp2((codes - 127).double()).unsqueeze(-1)
    return torch.where((codes == 255).unsqueeze(-1), torch.zeros_like(v), v).flatten(-2)


def quantize(x, format):
    """(values, scale codes) of x (..., D), float64 and int64"""
    codes = scale_codes(x, format)
    return nearest(divide(x, codes), format), codes


def values(codes):
    """What kept codes stand for before their scale, float64: uint8 holds e2m1 pairs"""
    codes = codes.cpu()
    if codes.dtype != torch.uint8:
        return codes.float().double()
    pair = torch.stack((codes & 15, codes >> 4), -1).long().flatten(-2)
    return torch.where(pair >= 8, -1.0, 1.0).double() * E2M1[pair & 7]


def byte(scales):
    return scales.cpu().view(torch.uint8).long()


def decode(codes, scales):
    """float64 values with their scales"""
    b = byte(scales)
    s = torch.where(b == 255, float("nan"), torch.exp2((b - 127).double()))
    return (values(codes).unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def pack(q):
    """uint8 pairs of e2m1 values q"""
    idx = torch.searchsorted(E2M1, q.abs().double().contiguous())
    code = (idx + 8 * torch.signbit(q).long()).to(torch.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4


def kept(x, format):
    """(codes, scales) as they are kept, on the CPU, of float values x"""
    q, b = quantize(x, format)
    codes = pack(q) if format == "e2m1" else q.to(torch.float8_e4m3fn)
    return codes, b.to(torch.uint8).view(torch.float8_e8m0fnu)
