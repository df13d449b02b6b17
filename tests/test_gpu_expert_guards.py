"""Rows by expert through the C ABI, each buffer that a call writes in the middle of a larger one: what lies on either side
stays as it was.  The sort with no assignment and around each number of workgroups, its workspace of the size that is asked
for."""
import ctypes
import os

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "mask_loss_amd", "libmask_loss_hip.so")
GUARD = 1 << 16  # bytes on either side


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.zeros(1, device="cuda")  # the HIP runtime is up before the library's first call
    so = ctypes.CDLL(LIB)
    vp, i64, sz = ctypes.c_void_p, ctypes.c_int64, ctypes.c_size_t
    so.ml_sort_by_expert_workspace_size.argtypes = [i64, i64, i64]
    so.ml_sort_by_expert_workspace_size.restype = sz
    so.ml_sort_by_expert.argtypes = [vp, i64, i64, i64, vp, vp, vp, vp, sz, vp]
    i32 = ctypes.c_int
    so.ml_to_experts.argtypes = [vp, i64, i64, i64, vp, vp, i64, vp, vp]
    so.ml_from_experts_forward.argtypes = [i32, i32, vp, vp, i64, i64, i64, vp, vp, i64, vp, vp]
    so.ml_from_experts_backward.argtypes = [i32, i32, vp, vp, vp, i64, i64, i64, vp, vp, i64, vp, vp, vp]
    return so


class Room:
    """`bytes` bytes between two guards, all of them 0xA5."""

    def __init__(self, bytes):
        self.bytes = bytes
        self.all = torch.full((bytes + 2 * GUARD,), 0xA5, dtype=torch.uint8, device="cuda")

    @property
    def ptr(self):
        return ctypes.c_void_p(self.all.data_ptr() + GUARD)

    def view(self, dtype, *shape):
        return self.all[GUARD:GUARD + self.bytes].view(dtype).view(*shape)

    def whole(self):
        sides = torch.cat([self.all[:GUARD], self.all[GUARD + self.bytes:]])
        return bool((sides == 0xA5).all())


def stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def plan(ids, experts):
    flat = np.where((ids < 0) | (ids >= experts), experts, ids).reshape(-1)
    order = np.argsort(flat, kind="stable")
    slots = np.empty_like(order)
    slots[order] = np.arange(len(order))
    return order, slots, np.searchsorted(flat[order], np.arange(experts + 1), side="left")


@pytest.mark.parametrize("experts", [4, 1023, 1024, 4000])
@pytest.mark.parametrize("tokens,k", [(0, 2), (5, 0), (0, 0), (1, 1), (1024, 1), (1025, 1), (4097, 1)])
def test_sort_stays_in_its_workspace(lib, tokens, k, experts):
    n = tokens * k
    ids = np.random.default_rng(n + experts).integers(-1, experts + 1, (tokens, k))
    given = torch.from_numpy(ids).cuda()
    ws = Room(lib.ml_sort_by_expert_workspace_size(tokens, k, experts))
    outs = [Room(8 * n), Room(8 * n), Room(8 * (experts + 1))]
    rc = lib.ml_sort_by_expert(ctypes.c_void_p(given.data_ptr()), tokens, k, experts, *[o.ptr for o in outs], ws.ptr, ws.bytes,
                               stream())
    torch.cuda.synchronize()
    assert rc == 0 and ws.whole() and all(o.whole() for o in outs)
    for o, want, name in zip(outs, plan(ids, experts), ("order", "slots", "offsets")):
        assert np.array_equal(o.view(torch.int64, -1).cpu().numpy(), want), name


@pytest.mark.parametrize("experts", [1, 1023, 1024, 4000])
@pytest.mark.parametrize("tokens,k", [(0, 2), (5, 0), (0, 0)])
def test_no_assignments(tokens, k, experts):
    from mask_loss_amd.functions import from_experts, sort_by_expert, to_experts
    order = sort_by_expert(torch.zeros(tokens, k, dtype=torch.int64, device="cuda"), experts)
    assert order.order.shape == (0,) and order.slots.shape == (tokens, k)
    assert order.offsets.shape == (experts + 1,) and not order.offsets.any()
    rows = to_experts(torch.randn(tokens, 24, device="cuda"), order)
    assert rows.shape == (0, 24) and not from_experts(rows, order).any()


def ptr(t):
    return ctypes.c_void_p(t.data_ptr())


# lanes to a row: 16, 64 and 256; whole and cut 16-byte chunks
@pytest.mark.parametrize("D", [32, 7, 260, 257, 1031])
@pytest.mark.parametrize("end,kept", [(6, 6), (2 ** 62, 6), (4, 4), (1, 1), (0, 0), (-5, 0)])
def test_places_outside(lib, end, kept, D):
    """Places outside the kept ones, and an end outside the rows: rows, sums and gradients of the kept places that slots name, zeros
    in the dropped places and for the dropped assignments, kept places that no slot names as they were, and nothing written
    outside (sums of one float32 product: exact)."""
    gen = torch.Generator().manual_seed(D + kept)
    slots = np.array([[0, 6], [-1, 2 ** 62], [1, -2 ** 63]])
    s, offsets = torch.from_numpy(slots).cuda(), torch.tensor([0, end], device="cuda")
    x, y, dout, w = (torch.randn(*shape, generator=gen) for shape in ((3, D), (6, D), (3, D), (3, 2)))
    xd, yd, gd, wd = (t.cuda() for t in (x, y, dout, w))
    rows, out, drows, dw = Room(6 * D * 4), Room(3 * D * 4), Room(6 * D * 4), Room(6 * 4)
    before = rows.view(torch.int32, 6, D).cpu()
    assert lib.ml_to_experts(ptr(xd), 3, 2, D * 4, ptr(s), ptr(offsets), 1, rows.ptr, stream()) == 0
    assert lib.ml_from_experts_forward(0, 0, ptr(yd), ptr(wd), 3, 2, D, ptr(s), ptr(offsets), 1, out.ptr, stream()) == 0
    assert lib.ml_from_experts_backward(0, 0, ptr(gd), ptr(yd), ptr(wd), 3, 2, D, ptr(s), ptr(offsets), 1, drows.ptr, dw.ptr,
                                        stream()) == 0
    torch.cuda.synchronize()
    assert all(r.whole() for r in (rows, out, drows, dw))
    want_rows, want_drows = before.clone(), before.clone()
    want_rows[kept:], want_drows[kept:] = 0, 0
    want_out, want_dw, bound = torch.zeros(3, D), torch.zeros(3, 2, dtype=torch.float64), torch.zeros(3, 2, dtype=torch.float64)
    for t in range(3):
        for j in range(2):
            p = int(slots[t, j])
            if not 0 <= p < kept:
                continue
            want_rows[p] = x[t].view(torch.int32)
            want_drows[p] = (w[t, j] * dout[t]).view(torch.int32)
            want_out[t] = w[t, j] * y[p]
            want_dw[t, j] = (dout[t].double() * y[p].double()).sum()
            bound[t, j] = (D / 16 + 8) * 2.0 ** -24 * (dout[t].double() * y[p].double()).abs().sum()
    assert torch.equal(rows.view(torch.int32, 6, D).cpu(), want_rows)
    assert torch.equal(drows.view(torch.int32, 6, D).cpu(), want_drows)
    assert torch.equal(out.view(torch.float32, 3, D).cpu(), want_out)
    assert bool(((dw.view(torch.float32, 3, 2).cpu().double() - want_dw).abs() <= bound + 2.0 ** -24 * want_dw.abs()).all())
