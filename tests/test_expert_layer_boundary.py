"""CPU checks of the boundary of the operators around the head's grouped products (root-mean-square norm, rows by expert,
microscaled values and products): the C ABI refuses bad arguments before it touches the GPU, with a code and a message; sizes
of workspaces; host tensors, wrong shapes, tangents and gradients of quantised values are refused."""
import ctypes
import os

import pytest

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "mask_loss_amd", "libmask_loss_hip.so")
EINVAL, EWORKSPACE, EUNSUPPORTED = 1, 2, 4
F32, BF16, F16 = 0, 1, 2
E2M1, E4M3 = 0, 1
PTR = ctypes.c_void_p(4096)  # never read: every call below is refused first
ODD = ctypes.c_void_p(4098)


class Shape(ctypes.Structure):
    _fields_ = [(k, ctypes.c_int64) for k in ["rows", "K", "N", "groups", "matrices"]]


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(LIB):
        pytest.skip("library not built")
    so = ctypes.CDLL(LIB)
    vp, i64, i32, sz, fl = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_size_t, ctypes.c_float
    so.ml_last_error.restype = ctypes.c_char_p
    so.ml_rms_norm_forward.argtypes = [i32, i32, vp, vp, vp, i64, i64, fl, vp, vp, vp, vp]
    so.ml_rms_norm_mx_forward.argtypes = [i32, i32, vp, vp, vp, i64, i64, fl, i32, vp, vp, vp, vp]
    so.ml_rms_norm_backward.argtypes = [i32, i32, vp, vp, vp, vp, vp, i64, i64, vp, vp, vp, sz, vp]
    so.ml_rms_norm_backward_workspace_size.argtypes = [i64, i64]
    so.ml_mx_quantize.argtypes = [i32, vp, i64, i64, i32, vp, vp, vp]
    so.ml_grouped_matmul_mx_workspace_size.argtypes = [ctypes.POINTER(Shape), i32, i32, i32]
    so.ml_grouped_matmul_mx.argtypes = [ctypes.POINTER(Shape), i32, vp, vp, i32, vp, vp, vp, i32, vp, vp, sz, vp]
    so.ml_sort_by_expert_workspace_size.argtypes = [i64, i64, i64]
    so.ml_sort_by_expert.argtypes = [vp, i64, i64, i64, vp, vp, vp, vp, sz, vp]
    so.ml_to_experts.argtypes = [vp, i64, i64, i64, vp, vp, i64, vp, vp]
    so.ml_from_experts_forward.argtypes = [i32, i32, vp, vp, i64, i64, i64, vp, vp, i64, vp, vp]
    so.ml_from_experts_backward.argtypes = [i32, i32, vp, vp, vp, i64, i64, i64, vp, vp, i64, vp, vp, vp]
    for n in ("rms_norm_backward", "grouped_matmul_mx", "sort_by_expert"):
        getattr(so, "ml_%s_workspace_size" % n).restype = sz
    return so


def refused(lib, rc, code, words):
    assert rc == code, (rc, lib.ml_last_error())
    assert words in lib.ml_last_error().decode()


def norm(lib, dtype=BF16, pdtype=BF16, x=PTR, res=None, rows=4, width=64, eps=1e-6, s=None, y=PTR):
    return lib.ml_rms_norm_forward(dtype, pdtype, x, res, None, rows, width, eps, s, y, None, None)


def norm_mx(lib, dtype=BF16, pdtype=BF16, x=PTR, res=None, rows=4, width=64, eps=1e-6, format=E4M3, s=None, codes=PTR,
            scales=PTR):
    return lib.ml_rms_norm_mx_forward(dtype, pdtype, x, res, None, rows, width, eps, format, s, codes, scales, None)


@pytest.mark.parametrize("fn", [norm, norm_mx])
def test_rms_norm_refusals(lib, fn):
    refused(lib, fn(lib, dtype=7, pdtype=7), EINVAL, "unsupported dtype")
    refused(lib, fn(lib, pdtype=F16), EINVAL, "input's dtype or be float32")
    refused(lib, fn(lib, dtype=F32, pdtype=BF16), EINVAL, "input's dtype or be float32")
    refused(lib, fn(lib, width=0), EINVAL, "width must be positive")
    refused(lib, fn(lib, rows=-1), EINVAL, "rows must not be negative")
    refused(lib, fn(lib, eps=-1.0), EINVAL, "eps")
    refused(lib, fn(lib, eps=float("nan")), EINVAL, "eps")
    refused(lib, fn(lib, x=None), EINVAL, "null pointer")
    refused(lib, fn(lib, res=PTR), EINVAL, "residual and sum go together")
    refused(lib, fn(lib, s=PTR), EINVAL, "residual and sum go together")
    refused(lib, fn(lib, rows=1 << 40, width=1 << 30), EUNSUPPORTED, "too many elements")
    refused(lib, fn(lib, width=(1 << 26) + 32), EUNSUPPORTED, "too many elements")
    assert fn(lib, rows=0, x=None) == 0  # nothing to do


def test_rms_norm_mx_refusals(lib):
    refused(lib, norm(lib, y=None), EINVAL, "null pointer")
    refused(lib, norm_mx(lib, format=2), EINVAL, "unknown format")
    refused(lib, norm_mx(lib, width=48), EINVAL, "multiple of 32")
    refused(lib, norm_mx(lib, codes=None), EINVAL, "null pointer")
    refused(lib, norm_mx(lib, scales=None), EINVAL, "null pointer")
    for which in ("x", "codes"):
        refused(lib, norm_mx(lib, **{which: ODD}), EINVAL, "16-byte aligned")
    refused(lib, norm_mx(lib, res=ODD, s=PTR), EINVAL, "16-byte aligned")
    refused(lib, norm_mx(lib, res=PTR, s=ODD), EINVAL, "16-byte aligned")


def norm_back(lib, rows=4, width=64, g=PTR, s=PTR, rstd=PTR, dx=PTR, dw=None, ws=None, bytes=0):
    return lib.ml_rms_norm_backward(BF16, F32, g, None, s, None, rstd, rows, width, dx, dw, ws, bytes, None)


def test_rms_norm_backward_refusals(lib):
    size = lib.ml_rms_norm_backward_workspace_size(4, 64)
    assert size >= 64 * 4 and lib.ml_rms_norm_backward_workspace_size(0, 64) > 0
    assert lib.ml_rms_norm_backward_workspace_size(-1, 64) == 0 and lib.ml_rms_norm_backward_workspace_size(4, 0) == 0
    for which in ("g", "s", "rstd"):
        refused(lib, norm_back(lib, **{which: None}), EINVAL, "null pointer")
    refused(lib, norm_back(lib, dw=PTR), EWORKSPACE, "workspace too small")
    refused(lib, norm_back(lib, dw=PTR, ws=PTR, bytes=size - 1), EWORKSPACE, "workspace too small")
    refused(lib, norm_back(lib, rows=-2), EINVAL, "rows")
    assert norm_back(lib, dx=None) == 0  # no gradient asked for


def test_quantize_refusals(lib):
    def call(dtype=BF16, x=PTR, rows=4, width=64, format=E4M3, codes=PTR, scales=PTR):
        return lib.ml_mx_quantize(dtype, x, rows, width, format, codes, scales, None)
    refused(lib, call(dtype=3), EINVAL, "unsupported dtype")
    refused(lib, call(format=-1), EINVAL, "unknown format")
    refused(lib, call(width=33), EINVAL, "multiple of 32")
    refused(lib, call(rows=-1), EINVAL, "negative")
    refused(lib, call(width=-32), EINVAL, "negative")
    refused(lib, call(rows=1 << 40, width=1 << 30), EUNSUPPORTED, "too many elements")
    for which in ("x", "codes", "scales"):
        refused(lib, call(**{which: None}), EINVAL, "null pointer")
    for which in ("x", "codes"):
        refused(lib, call(**{which: ODD}), EINVAL, "16-byte aligned")
    assert call(rows=0, x=None) == 0 and call(width=0, x=None) == 0


def product(lib, fx=E4M3, x=PTR, sx=PTR, fw=E2M1, w=PTR, sw=PTR, offsets=PTR, dtype=BF16, y=PTR, ws=PTR, bytes=1 << 40, **shape):
    s = dict(rows=64, K=128, N=256, groups=4, matrices=2)
    s.update(shape)
    return lib.ml_grouped_matmul_mx(ctypes.byref(Shape(**s)), fx, x, sx, fw, w, sw, offsets, dtype, y, ws, bytes, None)


def product_size(lib, fx=E4M3, fw=E2M1, dtype=BF16, **shape):
    s = dict(rows=64, K=128, N=256, groups=4, matrices=2)
    s.update(shape)
    return lib.ml_grouped_matmul_mx_workspace_size(ctypes.byref(Shape(**s)), fx, fw, dtype)


def test_product_refusals(lib):
    refused(lib, product(lib, dtype=3), EINVAL, "unsupported dtype")
    refused(lib, product(lib, fx=2), EINVAL, "unknown format")
    refused(lib, product(lib, fw=-1), EINVAL, "unknown format")
    refused(lib, product(lib, K=48), EINVAL, "multiple of 32")
    for bad in (dict(rows=-1), dict(K=-32), dict(N=-3), dict(groups=0), dict(matrices=0), dict(groups=5),
                dict(groups=2, matrices=4), dict(matrices=-2)):
        refused(lib, product(lib, **bad), EINVAL, "invalid shape")
    refused(lib, product(lib, groups=4002), EUNSUPPORTED, "groups")
    refused(lib, product(lib, K=(1 << 22) + 32), EUNSUPPORTED, "4194304")
    refused(lib, product(lib, N=(1 << 22) + 1), EUNSUPPORTED, "4194304")
    refused(lib, product(lib, rows=1 << 31), EUNSUPPORTED, "rows")
    refused(lib, product(lib, offsets=None, rows=63), EINVAL, "equal groups")
    for which in ("x", "sx", "w", "sw", "y"):
        refused(lib, product(lib, **{which: None}), EINVAL, "null pointer")
    for which in ("x", "w"):
        refused(lib, product(lib, **{which: ODD}), EINVAL, "16-byte aligned")
    # 4,000 groups of a row by 2^17 column tiles: past a launch's 2^32 threads
    refused(lib, product(lib, rows=4000, K=32, N=1 << 22, groups=4000, matrices=4000), EUNSUPPORTED, "too many tiles")
    assert product(lib, rows=0, x=None, y=None) == 0 and product(lib, N=0, x=None, y=None) == 0
    # few tiles and a long reduction: parts of it need a workspace (the query says so before any call)
    for dtype, shape in ((BF16, dict(rows=200, K=1 << 16, N=256, groups=1, matrices=1)),
                         (F32, dict(rows=200, K=1 << 16, N=256, groups=1, matrices=1)),
                         (F32, dict(rows=8, K=1 << 16, N=256, groups=1, matrices=1))):
        assert product_size(lib, dtype=dtype, **shape) > 256
        refused(lib, product(lib, dtype=dtype, ws=None, **shape), EWORKSPACE, "workspace too small")
        refused(lib, product(lib, dtype=dtype, bytes=255, **shape), EWORKSPACE, "workspace too small")


def test_product_workspace(lib):
    for dtype in (F32, BF16, F16):
        for fx in (E2M1, E4M3):
            for fw in (E2M1, E4M3):
                for shape in (dict(), dict(rows=0), dict(K=0), dict(N=0)):
                    assert product_size(lib, fx, fw, dtype, **shape) >= 256
                # bounded however long the reduction: the ring's tiles, or 64 planes
                assert product_size(lib, fx, fw, dtype, K=1 << 22, rows=200) <= max(64 * 200 * 256 * 4, 512 * 65536) + 256
    assert product_size(lib, dtype=5) == 0 and product_size(lib, fx=7) == 0 and product_size(lib, groups=3) == 0
    assert product_size(lib, K=33) == 0


def test_expert_refusals(lib):
    def sort(ids=PTR, tokens=8, k=2, experts=4, order=PTR, slots=PTR, offsets=PTR, ws=PTR, bytes=1 << 40):
        return lib.ml_sort_by_expert(ids, tokens, k, experts, order, slots, offsets, ws, bytes, None)

    def to(x=PTR, tokens=8, k=2, row_bytes=64, slots=PTR, offsets=PTR, experts=4, rows=PTR):
        return lib.ml_to_experts(x, tokens, k, row_bytes, slots, offsets, experts, rows, None)

    def back(dtype=BF16, wdtype=F32, rows=PTR, w=PTR, tokens=8, k=2, width=64, slots=PTR, offsets=PTR, experts=4, out=PTR):
        return lib.ml_from_experts_forward(dtype, wdtype, rows, w, tokens, k, width, slots, offsets, experts, out, None)

    def grad(dtype=BF16, wdtype=F32, g=PTR, rows=PTR, w=PTR, tokens=8, k=2, width=64, slots=PTR, offsets=PTR, experts=4, dr=PTR,
             dw=PTR):
        return lib.ml_from_experts_backward(dtype, wdtype, g, rows, w, tokens, k, width, slots, offsets, experts, dr, dw, None)

    for fn in (sort, to, back, grad):
        refused(lib, fn(tokens=-1), EINVAL, "must not be negative")
        refused(lib, fn(k=-1), EINVAL, "must not be negative")
        refused(lib, fn(experts=0), EINVAL, "at least one expert")
        refused(lib, fn(experts=4001), EUNSUPPORTED, "at most 4000")
        refused(lib, fn(tokens=1 << 30, k=2), EUNSUPPORTED, "assignments")
        refused(lib, fn(tokens=1 << 40, k=1 << 40), EUNSUPPORTED, "assignments")
        refused(lib, fn(offsets=None), EINVAL, "null pointer")
        refused(lib, fn(slots=None), EINVAL, "null pointer")
    refused(lib, sort(ids=None), EINVAL, "null pointer")
    refused(lib, sort(order=None), EINVAL, "null pointer")
    big = dict(tokens=4097, k=1, experts=200)
    size = lib.ml_sort_by_expert_workspace_size(4097, 1, 200)
    assert size > 256 and lib.ml_sort_by_expert_workspace_size(8, 2, 4) == 256
    assert lib.ml_sort_by_expert_workspace_size(-1, 2, 4) == 0 and lib.ml_sort_by_expert_workspace_size(8, 2, 0) == 0
    refused(lib, sort(ws=None, **big), EWORKSPACE, "workspace too small")
    refused(lib, sort(bytes=size - 1, **big), EWORKSPACE, "workspace too small")
    refused(lib, to(row_bytes=-1), EINVAL, "row_bytes")
    refused(lib, to(row_bytes=1 << 60), EUNSUPPORTED, "too many elements")
    refused(lib, to(x=None), EINVAL, "null pointer")
    refused(lib, to(rows=None), EINVAL, "null pointer")
    assert to(tokens=0, x=None) == 0 and to(k=0, x=None) == 0 and to(row_bytes=0, x=None) == 0
    for fn in (back, grad):
        refused(lib, fn(dtype=3, wdtype=3), EINVAL, "unsupported dtype")
        refused(lib, fn(wdtype=F16), EINVAL, "rows' dtype or be float32")
        refused(lib, fn(width=-1), EINVAL, "width")
        refused(lib, fn(width=1 << 60), EUNSUPPORTED, "too many elements")
        refused(lib, fn(rows=None), EINVAL, "null pointer")
    refused(lib, back(out=None), EINVAL, "null pointer")
    refused(lib, grad(g=None), EINVAL, "null pointer")
    assert back(tokens=0, rows=None) == 0 and back(width=0, rows=None) == 0
    assert grad(dr=None, dw=None) == 0 and grad(k=0, g=None) == 0


def test_host_tensors_and_shapes():
    from mask_loss_amd.functions import (ExpertOrder, from_experts, grouped_matmul_mx, mx_quantize, rms_norm, rms_norm_mx,
                                         sort_by_expert, to_experts)
    x, w = torch.zeros(4, 64), torch.ones(64)
    slots, offsets = torch.zeros(4, 2, dtype=torch.int64), torch.tensor([0, 8])
    order = ExpertOrder(slots.flatten(), slots, offsets)
    for grad in (False, True):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            rms_norm(x.clone().requires_grad_(grad), w, residual=x)
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            to_experts(x.clone().requires_grad_(grad), order)
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            from_experts(torch.zeros(8, 64).requires_grad_(grad), order, torch.ones(4, 2))
    codes, scales = torch.zeros(4, 64, dtype=torch.float8_e4m3fn), torch.zeros(4, 2, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    wc, ws = torch.zeros(1, 8, 32, dtype=torch.uint8), torch.zeros(1, 8, 2, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    for call in (lambda: rms_norm_mx(x, w), lambda: mx_quantize(x), lambda: sort_by_expert(slots, 3),
                 lambda: grouped_matmul_mx(codes, scales, wc, ws, torch.tensor([0, 4]))):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()
    for bad in ("e5m2", "", "E4M3"):
        with pytest.raises(ValueError, match="format must be"):
            mx_quantize(x, bad)
        with pytest.raises(ValueError, match="format must be"):
            rms_norm_mx(x, w, format=bad)


def test_gradients_of_quantised_values_are_refused():
    from mask_loss_amd.functions import mx_quantize, rms_norm_mx
    x, w = torch.zeros(4, 64), torch.ones(64)
    leaf = x.clone().requires_grad_(True)
    for call in (lambda: mx_quantize(leaf), lambda: rms_norm_mx(leaf, w), lambda: rms_norm_mx(x, w.clone().requires_grad_(True)),
                 lambda: rms_norm_mx(x, w, residual=leaf)):
        with pytest.raises(NotImplementedError, match="no gradient"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def test_tangents_are_refused():
    """A tensor that carries a tangent: every form raises, none leaves the tangent behind."""
    import mask_loss_amd
    from torch.autograd import forward_ad
    from mask_loss_amd.functions import ExpertOrder, from_experts, mx_quantize, rms_norm, rms_norm_mx, to_experts
    ml = mask_loss_amd.mask_loss
    x, w, stat = torch.ones(4, 64), torch.ones(64), torch.ones(4)
    slots, offsets = torch.zeros(4, 2, dtype=torch.int64), torch.tensor([0, 8])
    order = ExpertOrder(slots.flatten(), slots, offsets)
    y, g = torch.ones(8, 64), torch.ones(4, 2)
    calls = [(lambda a, b, c: rms_norm(a, b, 1e-6, c), (x, w, x)), (lambda a, b, c: rms_norm_mx(a, b, 1e-6, c), (x, w, x)),
             (mx_quantize, (x,)), (lambda a: to_experts(a, order), (x,)), (lambda a, b: from_experts(a, order, b), (y, g)),
             (lambda a, b, c, d, e: ml.rms_norm_backward(a, b, c, d, e), (x, x, x, w, stat)),
             (lambda a, b, c: ml.from_experts_backward(a, b, slots, offsets, c), (x, y, g))]
    with forward_ad.dual_level():
        for fn, args in calls:
            for i in range(len(args)):
                for grad in (False, True):
                    these = [t.clone() for t in args]
                    these[i] = forward_ad.make_dual(these[i], torch.ones_like(these[i]))
                    if grad:
                        these[0].requires_grad_(True)
                    with pytest.raises(NotImplementedError, match="forward-mode|no gradient"):
                        fn(*these)


@pytest.mark.parametrize("experts", [1, 4, 1023, 1024, 4000])
@pytest.mark.parametrize("tokens,k", [(0, 2), (5, 0), (0, 0), (1, 1), (1024, 1), (1025, 1), (4096, 1), (4097, 1), (70001, 3)])
def test_sort_workspace_holds_totals_and_counts(lib, tokens, k, experts):
    """Several workgroups keep totals and a row of counts for each 1,024 assignments, one row at least, also where there is no
    assignment: experts + 1 numbers of 4 bytes to a row.  One workgroup (4,096 assignments and 1,023 experts at most) needs none."""
    n, size = tokens * k, lib.ml_sort_by_expert_workspace_size(tokens, k, experts)
    if n <= 4096 and experts <= 1023:
        assert size == 256
    else:
        rows = 1 + max(1, -(-n // 1024))
        assert rows * (experts + 1) * 4 <= size <= rows * (experts + 1) * 4 + 255
