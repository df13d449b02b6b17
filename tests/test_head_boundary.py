"""CPU checks of the layer norm's, grouped products' and mask logits' boundary: the C
ABI refuses bad arguments before it touches the GPU, with a code and a message; sizes
of workspaces; host tensors and wrong shapes are rejected."""
import ctypes
import os

import pytest

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "mask_loss_amd", "libmask_loss_hip.so")
EINVAL, EWORKSPACE, EUNSUPPORTED = 1, 2, 4
F32, BF16, F16 = 0, 1, 2
PTR = ctypes.c_void_p(4096)  # never read: every call below is refused first


class Shape(ctypes.Structure):
    _fields_ = [(k, ctypes.c_int64) for k in ["rows", "K", "N", "groups", "matrices"]]


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(LIB):
        pytest.skip("library not built")
    so = ctypes.CDLL(LIB)
    vp, i64, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int
    so.ml_last_error.restype = ctypes.c_char_p
    so.ml_layer_norm_forward.argtypes = [i32, i32, vp, vp, vp, i64, i64, ctypes.c_float, vp, vp, vp, vp]
    so.ml_layer_norm_backward.argtypes = [i32, i32, vp, vp, vp, vp, vp, i64, i64, vp, vp, vp, vp, ctypes.c_size_t, vp]
    so.ml_layer_norm_backward_workspace_size.argtypes = [i64, i64]
    so.ml_layer_norm_backward_workspace_size.restype = ctypes.c_size_t
    so.ml_grouped_matmul_workspace_size.argtypes = [ctypes.POINTER(Shape), i32, i32]
    so.ml_grouped_matmul_workspace_size.restype = ctypes.c_size_t
    for n in ("forward", "backward_input", "backward_weight"):
        getattr(so, "ml_grouped_matmul_" + n).argtypes = [ctypes.POINTER(Shape), i32, vp, vp, i32, vp, vp, vp,
                                                          ctypes.c_size_t, vp]
    return so


def refused(lib, rc, code, words):
    assert rc == code, (rc, lib.ml_last_error())
    assert words in lib.ml_last_error().decode()


def norm(lib, dtype=BF16, pdtype=BF16, x=PTR, rows=4, width=64, eps=1e-5, y=PTR, mean=None, rstd=None):
    return lib.ml_layer_norm_forward(dtype, pdtype, x, None, None, rows, width, eps, y, mean, rstd, None)


def test_layer_norm_refusals(lib):
    refused(lib, norm(lib, dtype=7, pdtype=7), EINVAL, "unsupported dtype")
    refused(lib, norm(lib, pdtype=F16), EINVAL, "input's dtype or be float32")
    refused(lib, norm(lib, dtype=F32, pdtype=BF16), EINVAL, "input's dtype or be float32")
    refused(lib, norm(lib, width=0), EINVAL, "width must be positive")
    refused(lib, norm(lib, rows=-1), EINVAL, "rows must not be negative")
    refused(lib, norm(lib, eps=-1.0), EINVAL, "eps")
    refused(lib, norm(lib, eps=float("nan")), EINVAL, "eps")
    refused(lib, norm(lib, x=None), EINVAL, "null pointer")
    refused(lib, norm(lib, y=None), EINVAL, "null pointer")
    refused(lib, norm(lib, mean=PTR), EINVAL, "mean and rstd go together")
    refused(lib, norm(lib, rows=1 << 40, width=1 << 30), EUNSUPPORTED, "too many elements")
    refused(lib, norm(lib, width=1 << 32), EUNSUPPORTED, "too many elements")
    refused(lib, norm(lib, width=(1 << 26) + 1), EUNSUPPORTED, "too many elements")
    assert norm(lib, rows=0, x=None, y=None) == 0  # nothing to do


def norm_back(lib, rows=4, width=64, g=PTR, x=PTR, mean=PTR, rstd=PTR, dx=PTR, dw=None, db=None, ws=None, bytes=0):
    return lib.ml_layer_norm_backward(BF16, F32, g, x, None, mean, rstd, rows, width, dx, dw, db, ws, bytes, None)


def test_layer_norm_backward_refusals(lib):
    size = lib.ml_layer_norm_backward_workspace_size(4, 64)
    assert size >= 2 * 64 * 4
    assert lib.ml_layer_norm_backward_workspace_size(-1, 64) == 0
    assert lib.ml_layer_norm_backward_workspace_size(4, 0) == 0
    assert lib.ml_layer_norm_backward_workspace_size(0, 64) > 0
    for g in ("g", "x", "mean", "rstd"):
        refused(lib, norm_back(lib, **{g: None}), EINVAL, "null pointer")
    # (a call that were not refused would end at the missing device here, not at these pointers)
    refused(lib, norm_back(lib, dw=PTR), EWORKSPACE, "workspace too small")
    refused(lib, norm_back(lib, db=PTR, ws=PTR, bytes=size - 1), EWORKSPACE, "workspace too small")
    refused(lib, norm_back(lib, rows=-2), EINVAL, "rows")
    assert norm_back(lib, dx=None) == 0  # no gradient asked for


def grouped(lib, name="forward", dtype=BF16, x=PTR, w=PTR, offsets=PTR, out=PTR, ws=PTR, bytes=1 << 40, **shape):
    s = dict(rows=64, K=128, N=256, groups=4, matrices=2)
    s.update(shape)
    fn = getattr(lib, "ml_grouped_matmul_" + name)
    return fn(ctypes.byref(Shape(**s)), dtype, x, w, 0, offsets, out, ws, bytes, None)


def size_of(lib, dtype=BF16, product=0, **shape):
    s = dict(rows=64, K=128, N=256, groups=4, matrices=2)
    s.update(shape)
    return lib.ml_grouped_matmul_workspace_size(ctypes.byref(Shape(**s)), dtype, product)


@pytest.mark.parametrize("name", ["forward", "backward_input", "backward_weight"])
def test_grouped_refusals(lib, name):
    refused(lib, grouped(lib, name, dtype=3), EINVAL, "unsupported dtype")
    for bad in (dict(rows=-1), dict(K=-1), dict(N=-3), dict(groups=0), dict(matrices=0), dict(groups=5),
                dict(groups=2, matrices=4), dict(matrices=-2)):
        refused(lib, grouped(lib, name, **bad), EINVAL, "invalid shape")
    refused(lib, grouped(lib, name, groups=4002), EUNSUPPORTED, "groups")
    refused(lib, grouped(lib, name, K=(1 << 22) + 1), EUNSUPPORTED, "4194304")
    refused(lib, grouped(lib, name, N=(1 << 22) + 1), EUNSUPPORTED, "4194304")
    refused(lib, grouped(lib, name, rows=1 << 31), EUNSUPPORTED, "rows")
    refused(lib, grouped(lib, name, offsets=None, rows=63), EINVAL, "equal groups")
    refused(lib, grouped(lib, name, x=None), EINVAL, "null pointer")
    refused(lib, grouped(lib, name, w=None), EINVAL, "null pointer")
    refused(lib, grouped(lib, name, out=None), EINVAL, "null pointer")
    # few tiles and a long reduction: parts of it need a workspace (the query says so before any call)
    long = {"forward": dict(K=65536, N=256), "backward_input": dict(K=256, N=65536),
            "backward_weight": dict(rows=1 << 16, K=32, N=32)}[name]
    product = ["forward", "backward_input", "backward_weight"].index(name)
    assert size_of(lib, product=product, **long) > 256
    refused(lib, grouped(lib, name, ws=None, **long), EWORKSPACE, "workspace too small")
    refused(lib, grouped(lib, name, bytes=255, **long), EWORKSPACE, "workspace too small")
    # 4,000 groups of a row or matrices of a row by 32,768 column tiles: past a launch's 2^32 threads
    many = {"forward": dict(rows=4000, K=1, N=1 << 22), "backward_input": dict(rows=4000, K=1 << 22, N=1),
            "backward_weight": dict(rows=4000, K=1, N=1 << 22)}[name]
    refused(lib, grouped(lib, name, groups=4000, matrices=4000, **many), EUNSUPPORTED, "too many tiles")
    assert grouped(lib, name, K=0, N=0, x=None, w=None, out=None) == 0  # nothing to write


def test_grouped_workspace(lib):
    def size(*a, **kw):
        return size_of(lib, *a, **kw)

    for dtype in (F32, BF16, F16):
        for product in (0, 1, 2):
            assert size(dtype, product) >= 256
            assert size(dtype, product, rows=0) >= 256
            assert size(dtype, product, K=0, N=0) >= 256
    assert size(product=3) == 0 and size(product=-1) == 0 and size(dtype=9) == 0
    assert size(groups=3) == 0 and size(matrices=0) == 0 and size(K=1 << 23) == 0
    # bounded however long the reduction: 256 compute units' tiles, or 64 planes
    assert size(K=1 << 22, rows=200) <= max(64 * 200 * 256 * 4, 256 * 65536 * 4) + 256


def test_extension_refusals():
    import mask_loss_amd
    from mask_loss_amd.functions import grouped_matmul, layer_norm, mask_logits
    ml = mask_loss_amd.mask_loss
    x = torch.zeros(4, 8)
    for grad in (False, True):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            layer_norm(x.clone().requires_grad_(grad), torch.ones(8), torch.zeros(8))
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            grouped_matmul(x.clone().requires_grad_(grad), torch.zeros(2, 8, 3), torch.tensor([0, 2, 4]))
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            mask_logits(torch.zeros(1, 2, 4, 8).requires_grad_(grad), torch.zeros(2, 8, 5, 5))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ml.layer_norm_backward(x, x, None, torch.zeros(4), torch.zeros(4))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ml.grouped_matmul_backward_input(torch.zeros(4, 3), torch.zeros(2, 8, 3), torch.tensor([0, 2, 4]))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        ml.grouped_matmul_backward_weight(x, torch.zeros(4, 3), torch.tensor([0, 2, 4]), 2)


def test_mask_logits_shapes():
    from mask_loss_amd.functions import mask_logits
    f = torch.zeros(2, 8, 5, 5)
    for q, feat, o, words in ((torch.zeros(1, 2, 4, 8), torch.zeros(2, 8, 25), None, "features must be"),
                              (torch.zeros(1, 2, 4, 7), f, None, "queries must be"),
                              (torch.zeros(2, 4, 8), f, None, "queries must be"),
                              (torch.zeros(1, 3, 4, 8), f, None, "same batch size"),
                              (torch.zeros(1, 2, 4, 8), f, torch.tensor([0, 1, 2]), "with offsets"),
                              (torch.zeros(6, 8), f, torch.tensor([0, 6]), "offsets must have shape")):
        for grad in (False, True):
            with pytest.raises(ValueError, match=words):
                mask_logits(q.clone().requires_grad_(grad), feat, o)
