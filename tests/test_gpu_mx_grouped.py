"""Products of microscaled operands on the GPU against float64: formats, dtypes, sizes on both sides of the tiles and
steps, groups of every kind, NaN scales and the scales' extremes.

Tolerances, with u = 2^-24 and p the products behind a result:

* at most K additions in float32: K u sum |p|;
* a 16-bit result with an e4m3 operand loses, in eight neighbours of the reduced index, less than 2^-13 of the largest product
  for each of the other seven: 2^-10 of the sum of the eights' largest products more.  Operands whose e4m3 values span four
  binades lose nothing (a product's last bit is 6 + 6 below the largest's leading one), e2m1 ones neither;
* half a step of the result's dtype: 2^-8 (bfloat16), 2^-11 (float16) or 2^-24 of its value.
"""
import pytest

torch = pytest.importorskip("torch")

import mx_reference as mx  # noqa: E402

pytestmark = pytest.mark.gpu

TDT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
U = 2.0 ** -24
PAIRS = [("e4m3", "e2m1"), ("e2m1", "e2m1"), ("e4m3", "e4m3"), ("e2m1", "e4m3")]


@pytest.fixture(scope="module", autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def operand(shape, format, seed, few_binades=False, scales=(117, 131)):
    """(codes, scales) on the CPU: any codes but NaN, or e4m3 of four binades"""
    gen = torch.Generator().manual_seed(seed)
    rows, K = shape[:-1], shape[-1]
    if format == "e2m1":
        codes = torch.randint(0, 256, (*rows, K // 2), generator=gen).to(torch.uint8)
    else:
        raw = torch.randint(5 << 3 if few_binades else 0, 9 << 3 if few_binades else 127, (*rows, K), generator=gen)
        raw = raw + 128 * torch.randint(0, 2, raw.shape, generator=gen)
        codes = raw.to(torch.uint8).view(torch.float8_e4m3fn)
    b = torch.randint(scales[0], scales[1], (*rows, K // 32), generator=gen).to(torch.uint8)
    return codes, b.view(torch.float8_e8m0fnu)


def quantized(shape, format, seed):
    """(codes, scales) of normal values, a few channels larger"""
    gen = torch.Generator().manual_seed(seed)
    return mx.kept(torch.randn(shape, generator=gen) * torch.exp(torch.randn(shape[-1], generator=gen)), format)


def edges(offsets, rows):
    out, last = [], 0
    for o in offsets:
        last = max(last, min(max(int(o), 0), rows))
        out.append(last)
    return out


def call(x, w, offsets, dtype):
    from mask_loss_amd.functions import grouped_matmul_mx
    return grouped_matmul_mx(x[0].cuda(), x[1].cuda(), w[0].cuda(), w[1].cuda(),
                             None if offsets is None else torch.tensor(offsets, device="cuda"), dtype)


def compare(x, w, offsets, dtype, drops):
    """drops: whether the instruction may drop bits of products"""
    y = call(x, w, offsets, dtype)
    assert y.dtype == dtype
    xv, wv = mx.decode(*x), mx.decode(*w)
    K, N, M = xv.shape[-1], wv.shape[1], wv.shape[0]
    groups = [xv[g] for g in range(xv.shape[0])] if offsets is None else None
    got = y.reshape(-1, N).double().cpu()
    rows = got.shape[0]
    if offsets is None:
        e = [g * xv.shape[1] for g in range(len(groups) + 1)]
        xv = xv.reshape(-1, K)
    else:
        e = edges(offsets, rows)
    want, bound = torch.zeros(rows, N, dtype=torch.float64), torch.zeros(rows, N, dtype=torch.float64)
    for g, (lo, hi) in enumerate(zip(e, e[1:])):
        a, b = xv[lo:hi], wv[g % M].t()
        want[lo:hi] = a @ b
        bound[lo:hi] = K * U * (a.abs() @ b.abs())
        if drops and hi > lo:
            eights = (a.view(hi - lo, K // 8, 8, 1).abs() * b.reshape(1, K // 8, 8, N).abs()).amax(2).sum(1)
            bound[lo:hi] += 2.0 ** -10 * eights
    tol = bound + STEP[dtype] * want.abs() * (1 + 2 ** -7) + (2.0 ** -25 if dtype == torch.float16 else 0.0) + 1e-37
    err = (got - want).abs()
    assert not bool((~(err <= tol)).any()), float((err / tol).max())
    return y


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("fx,fw", PAIRS)
@pytest.mark.parametrize("K", [32, 64, 96, 128, 160, 224, 256, 288, 512, 1056, 2048])
@pytest.mark.parametrize("rows,N,offsets", [(20, 40, [0, 7, 7, 20]), (75, 70, [0, 30, 33, 75]), (300, 129, [0, 131, 150, 300])])
def test_exact_products(dt, fx, fw, K, rows, N, offsets):
    """Products that no format drops bits of: few rows to a group, and many."""
    x, w = operand((rows, K), fx, K, True, (125, 130)), operand((3, N, K), fw, K + 1, True, (125, 130))
    compare(x, w, offsets, TDT[dt], False)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("fx,fw", PAIRS)
@pytest.mark.parametrize("rows,N,K,offsets", [(33, 70, 320, [0, 30, 33]), (200, 257, 640, [3, 100, 190])])
def test_normal_values(dt, fx, fw, rows, N, K, offsets):
    x, w = quantized((rows, K), fx, 3), quantized((2, N, K), fw, 4)
    drops = dt != "f32" and "e4m3" in (fx, fw)
    y = compare(x, w, offsets, TDT[dt], drops)
    # what is dropped is far less than its bound: 1e-4 of the result's size
    xv, wv = mx.decode(*x), mx.decode(*w)
    want = torch.zeros(rows, N, dtype=torch.float64)
    for g in range(2):
        want[offsets[g]:offsets[g + 1]] = xv[offsets[g]:offsets[g + 1]] @ wv[g].t()
    off = float((y.double().cpu() - want).norm() / want.norm())
    assert off <= (1e-4 if drops else 1e-6) + STEP[TDT[dt]]


# K: any blocks, whole 128 and whole 512, which have kernels of their own
@pytest.mark.parametrize("K", [192, 384, 512])
@pytest.mark.parametrize("fx,fw", PAIRS)
@pytest.mark.parametrize("N", [1, 2, 3, 5, 15, 16, 17, 64, 127, 128, 130, 255, 384, 1000])
def test_columns(fx, fw, N, K):
    for rows, offsets in ((9, [0, 4, 9]), (150, [0, 70, 150])):
        x, w = operand((rows, K), fx, N, True, (125, 130)), operand((2, N, K), fw, N + 1, True, (125, 130))
        for dtype in (torch.bfloat16, torch.float32):
            compare(x, w, offsets, dtype, False)


GROUPS = [([0, 1], 1, 1), ([0, 0, 1], 1, 2), ([0, 0, 0, 0], 5, 3), ([2, 5, 9], 12, 2), ([0, 128, 256], 256, 2),
          ([0, 129, 257, 300], 310, 3), ([5, 3, 40, 20, 60], 50, 4), ([-4, 10, 2 ** 40], 33, 2), ([0, 40, 80, 120, 160], 170, 2),
          ([10, 60, 61, 61, 150, 200, 333], 340, 3), ([0] + [1] * 40, 3, 40), (list(range(65)), 64, 64), ([0, 500], 500, 1),
          ([0, 90, 90, 300, 420, 600, 600, 777, 900], 1000, 2), (list(range(0, 3001, 50)), 3010, 60)]


@pytest.mark.parametrize("K", [160, 256, 512])
@pytest.mark.parametrize("fx,fw", PAIRS)
@pytest.mark.parametrize("offsets,rows,M", GROUPS)
def test_groups(fx, fw, offsets, rows, M, K):
    """Empty groups, rows before the first and behind the last (zeros), borders that decrease or lie outside, groups
    that share a matrix, one group, many."""
    x, w = operand((rows, K), fx, rows, True, (125, 130)), operand((M, 72, K), fw, M, True, (125, 130))
    y = compare(x, w, offsets, torch.bfloat16, False)
    e = edges(offsets, rows)
    assert not y[:e[0]].any() and not y[e[-1]:].any()


@pytest.mark.parametrize("fx,fw", PAIRS)
@pytest.mark.parametrize("K", [96, 128, 1024])
@pytest.mark.parametrize("G,n,M", [(1, 1, 1), (4, 5, 2), (6, 100, 3), (3, 130, 3), (2, 0, 2)])
def test_equal_groups(fx, fw, G, n, M, K):
    x, w = operand((G, n, K), fx, 5, True, (125, 130)), operand((M, 50, K), fw, 6, True, (125, 130))
    compare(x, w, None, torch.float16, False)


@pytest.mark.parametrize("fx,fw", PAIRS)
@pytest.mark.parametrize("rows,K,N", [(3, 8192, 64), (40, 16384, 20), (200, 8224, 96), (200, 8192, 96), (200, 8192, 97),
                                      (130, 4224, 260), (300, 1024, 512)])
def test_split_reductions(fx, fw, rows, K, N):
    """Few tiles and long reductions, which are split and joined."""
    x, w = operand((rows, K), fx, 7, True, (125, 130)), operand((1, N, K), fw, 8, True, (125, 130))
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        compare(x, w, [0, rows], dtype, False)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("fx,fw", PAIRS)
@pytest.mark.parametrize("rows,M,offsets", [(50, 3, [2, 20, 31, 47]), (29, 2, [1, 9, 9, 20, 27]), (90, 3, [0, 31, 62, 90])])
@pytest.mark.parametrize("K", [16384 + 32, 8192])
def test_split_reductions_of_groups(dt, fx, fw, rows, M, offsets, K):
    """The same with few rows to a group: 16 and 32 rows to a tile, rows outside, groups that share a matrix, and
    columns and a last part of no round number."""
    x, w = operand((rows, K), fx, 7, True, (125, 130)), operand((M, 21, K), fw, 8, True, (125, 130))
    compare(x, w, offsets, TDT[dt], False)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("fx,fw", PAIRS)
@pytest.mark.parametrize("rows", [6, 140])
def test_scales(fx, fw, dt, rows):
    """The smallest and largest scales where their product is not, and NaN scales: a row's and a column's alone."""
    most = 246  # (e4m3 in a float32 result: 448 * 2^119 is finite, twice that is not)
    for lo, hi in ((0, 4), (most - 3, most + 1)):
        x = operand((rows, 128), fx, 9, True, (lo, hi))
        w = operand((1, 40, 128), fw, 10, True, (252 - hi, 256 - hi))
        x[1].view(torch.uint8)[0] = lo
        drops = False
        if lo == 0 and dt == "f32" and "e4m3" in (fx, fw):
            x[1].view(torch.uint8).clamp_(min=4)  # values below 2^-126 may count as zero
        compare(x, w, [0, rows], TDT[dt], drops)
    for K in (320, 384, 1024):
        x, w = operand((rows, K), fx, 11, True), operand((2, 40, K), fw, 12, True)
        offsets = [1, rows // 2, rows - 2]
        clean = call(x, w, offsets, TDT[dt])
        for t, at in ((x, (2, 9)), (x, (0, 0)), (x, (rows - 1, 5)), (w, (1, 7, 3))):
            b = t[1].view(torch.uint8).clone()
            b[at] = 255
            bad = (t[0], b.view(torch.float8_e8m0fnu))
            y = call(bad, w, offsets, TDT[dt]) if t is x else call(x, bad, offsets, TDT[dt])
            hit = torch.zeros_like(clean, dtype=torch.bool)
            if t is w:
                hit[offsets[1]:offsets[2], 7] = True
            elif offsets[0] <= at[0] < offsets[2]:
                hit[at[0]] = True
            assert bool(torch.isnan(y[hit]).all()) and torch.equal(y[~hit], clean[~hit])


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("fx,fw", PAIRS)
@pytest.mark.parametrize("rows,K,N,groups", [(3000, 512, 4096, 5), (2500, 640, 2056, 3), (16640, 128, 16640, 1),
                                             (16640, 512, 16640, 7)])
def test_many_tiles(fx, fw, dt, rows, K, N, groups):
    """Workgroups that make several tiles, and over 32 of them.  All scales 1 and few binades: every partial sum is
    a float32, so any order gives the same result, rounded once."""
    x, w = operand((rows, K), fx, 13, True, (127, 128)), operand((groups, N, K), fw, 14, True, (127, 128))
    gen = torch.Generator().manual_seed(15)
    cuts = torch.randint(0, rows + 1, (groups - 1,), generator=gen).sort().values.tolist()
    offsets = [0, *cuts, rows - 7]
    y = call(x, w, offsets, TDT[dt])
    xv, wv = (mx.values(t[0]).float().cuda() for t in (x, w))
    for g, (lo, hi) in enumerate(zip(edges(offsets, rows), edges(offsets, rows)[1:])):
        assert torch.equal(y[lo:hi], (xv[lo:hi] @ wv[g].t()).to(TDT[dt])), g
    assert not y[rows - 7:].any()


def test_no_size():
    x, w = operand((4, 64), "e4m3", 1), operand((2, 0, 64), "e2m1", 1)
    assert call(x, w, [0, 2, 4], torch.bfloat16).shape == (4, 0)
    x, w = operand((0, 64), "e4m3", 1), operand((2, 5, 64), "e2m1", 1)
    assert call(x, w, [0, 0, 0], torch.bfloat16).shape == (0, 5)
    x, w = operand((4, 0), "e4m3", 1), operand((2, 5, 0), "e2m1", 1)
    y = call(x, w, [0, 2, 4], torch.bfloat16)
    assert y.shape == (4, 5) and not y.any()
    for dtype in (torch.bfloat16, torch.float32):
        x, w = operand((300, 0), "e4m3", 1), operand((2, 5, 0), "e2m1", 1)
        y = call(x, w, [0, 100, 290], dtype)
        assert y.shape == (300, 5) and not y.any()


@pytest.mark.parametrize("each", [1, 40])
@pytest.mark.parametrize("matrices", [4000, 40])
def test_most_groups(each, matrices):
    """4,000 groups, the most: their borders fill much of the LDS."""
    rows, K, N = 4000 * each, 128, 24
    x, w = operand((rows, K), "e4m3", 3, True, (127, 128)), operand((matrices, N, K), "e2m1", 4, True, (127, 128))
    gen = torch.Generator().manual_seed(5)
    offsets = [0, *torch.randint(0, rows + 1, (3999,), generator=gen).sort().values.tolist(), rows]
    y = call(x, w, offsets, torch.float32)
    group = torch.searchsorted(torch.tensor(offsets[1:]), torch.arange(rows), right=True) % matrices
    xv, wv = mx.values(x[0]).float().cuda(), mx.values(w[0]).float().cuda()
    for lo in range(0, rows, 20000):  # every partial sum is a float32: any order
        part = group[lo:lo + 20000].cuda()
        assert torch.equal(y[lo:lo + 20000], (xv[lo:lo + 20000, None, :] * wv[part]).sum(-1))


def test_layouts():
    """Codes on no 16-byte boundary, transposed ones, scales on an odd byte."""
    from mask_loss_amd.functions import grouped_matmul_mx
    for K, rows in ((96, 40), (384, 150), (512, 150)):
        x, w = operand((rows, K), "e4m3", 2, True), operand((2, 24, K), "e2m1", 3, True)
        moves(grouped_matmul_mx, [t.cuda() for t in (*x, *w)], torch.tensor([0, 11, rows], device="cuda"))


def moves(fn, args, o):
    want = fn(*args, o)

    def odd(t):
        room = torch.empty(t.numel() + 1, dtype=torch.uint8, device="cuda")
        room[1:] = t.reshape(-1).view(torch.uint8)
        return room[1:].view(t.dtype).view(t.shape)

    for i in range(4):
        moved = list(args)
        moved[i] = odd(args[i])
        assert moved[i].data_ptr() % 16
        assert torch.equal(fn(*moved, o), want)
        moved[i] = args[i].view(torch.uint8).transpose(-1, -2).contiguous().transpose(-1, -2).view(args[i].dtype)
        assert torch.equal(fn(*moved, o), want)


def test_past_32_bits():
    """Operands and results of over 2^32 values: the last rows, columns and matrix as in calls of their own."""
    from mask_loss_amd.functions import grouped_matmul_mx
    gen = torch.Generator(device="cuda").manual_seed(3)
    R, K, N = 4200, 1 << 20, 40
    codes = torch.zeros(R, K // 2, dtype=torch.uint8, device="cuda")
    codes[-9:] = torch.randint(0, 256, (9, K // 2), generator=gen, device="cuda").to(torch.uint8)
    scales = torch.full((R, K // 32), 120, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    wc = torch.randint(0, 256, (1, N, K // 2), generator=gen, device="cuda").to(torch.uint8)
    ws = torch.full((1, N, K // 32), 120, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    o = torch.tensor([0, R], device="cuda")
    y = grouped_matmul_mx(codes, scales, wc, ws, o, torch.float32)
    few = grouped_matmul_mx(codes[-9:], scales[-9:], wc, ws, torch.tensor([0, 9], device="cuda"), torch.float32)
    # exact sums of e2m1 products: another order of float32 additions
    assert not y[:-9].any() and bool(((y[-9:] - few).abs() <= 2 * K * U * 36 * 2.0 ** -14 * K).all())
    assert float((y[-9:] - few).norm() / few.norm()) < 1e-5
    del codes, scales, wc, ws, y
    rows, M, N, K = 70000, 2, 65536, 64
    x = [t.cuda() for t in operand((rows, K), "e4m3", 4, True)]
    w = [t.cuda() for t in operand((M, N, K), "e2m1", 5, True)]
    y = grouped_matmul_mx(*x, *w, torch.tensor([0, 60000, rows], device="cuda"))
    tail = grouped_matmul_mx(x[0][-200:], x[1][-200:], w[0][1:], w[1][1:], torch.tensor([0, 200], device="cuda"))
    assert y.numel() > 1 << 32 and torch.equal(y[-200:], tail)


def test_refusals():
    from mask_loss_amd.functions import grouped_matmul_mx
    x, s = (t.cuda() for t in operand((4, 64), "e4m3", 1))
    w, ws = (t.cuda() for t in operand((2, 5, 64), "e2m1", 1))
    o = torch.tensor([0, 2, 4], device="cuda")
    for args, words in (((x, s, w, ws, o.int()), "int64"), ((x, s, w, ws, o[:1]), "offsets must have shape"),
                        ((x, s, w, ws, torch.tensor([0, 1, 2, 4], device="cuda")), "multiple of the number"),
                        ((x, s.view(torch.uint8), w, ws, o), "float8_e8m0fnu"), ((x, s[:, :1], w, ws, o), "whole blocks"),
                        ((x[:, :48], s, w, ws, o), "whole blocks"), ((x.float(), s, w, ws, o), "e2m1"),
                        ((x, s, w[0], ws[0], o), "matrices, N, K"), ((x, s, w[:, :, :16], ws[:, :, :1], o), "same K"),
                        ((x, s, w, ws, None), "without offsets"), ((x.cpu(), s, w, ws, o), "CUDA tensor"),
                        ((x, s, w.cpu(), ws, o), "CUDA tensor"), ((x, s, w, ws, o.cpu()), "CUDA tensor"),
                        ((x, s, w, ws, o, torch.float64), "dtype must be")):
        with pytest.raises(RuntimeError, match=words):
            grouped_matmul_mx(*args)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("fx,fw", [("e4m3", "e2m1"), ("e4m3", "e4m3"), ("e2m1", "e4m3")])
@pytest.mark.parametrize("rows,K", [(8, 512), (200, 512), (200, 128), (200, 160)])
def test_values_outside_bfloat16(rows, K, fx, fw, dt):
    """An e4m3 operand whose values with their scale lie outside bfloat16's normal range, and another that brings the products
    back: right in 16 bits, where the instruction applies both scales at once; in float32 the largest values are infinite from
    2^128 on and the smallest count as they are or as zero below 2^-126.  All values are equal: sums are exact."""
    def full(shape, format, value, scale):
        codes, _ = mx.kept(torch.full((*shape, K), value), format)
        return codes, torch.full((*shape, K // 32), scale, dtype=torch.uint8).view(torch.float8_e8m0fnu)

    which = "x" if fx == "e4m3" else "w"
    # (codes of 448, of 256 and, for a block of ones, of the format's last binade: 256 or 4)
    for value, scale, result in ((448.0, 254, "infinite"), (256.0, 246, "exact"), (256.0, 0, "exact"), (256.0, 0, "small")):
        other = 27 if scale > 127 else 227
        a = full((rows,), fx, value if which == "x" else 1.0, scale if which == "x" else other)
        b = full((1, 24), fw, value if which == "w" else 1.0, scale if which == "w" else other)
        if result == "small":  # the format's smallest value: 2^-9 2^-127
            t = a if which == "x" else b
            t[0].view(torch.uint8).fill_(1)
        y = call(a, b, [0, rows], TDT[dt]).double().cpu()
        want = mx.decode(*a) @ mx.decode(*b)[0].t()
        assert float(want.max()) == float(want.min()) and 2.0 ** -120 < float(want[0, 0]) < 2.0 ** 120
        near = (y - want).abs() <= STEP[TDT[dt]] * want
        if dt == "f32" and result == "infinite":
            assert bool(torch.isinf(y).all())
        elif dt == "f32" and result == "small":
            assert bool((near | (y == 0)).all()) and float(y.max()) == float(y.min())
        else:
            assert bool(near.all())
