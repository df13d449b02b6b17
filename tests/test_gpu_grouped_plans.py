"""The grouped products of grouped_plans.py on the GPU against float64: every tile of the ring kernel over
several stages and a cut last one, in each storage order, with groups that share a matrix or not, whole and in
parts.  Tolerance: test_gpu_grouped.py's."""
import pytest

torch = pytest.importorskip("torch")

import grouped_plans as gp
import test_gpu_grouped as base

pytestmark = pytest.mark.gpu

need_gpu = base.need_gpu


def reference(x, w, dy, edges, product, transposed):
    """(value, sum of |terms|, terms) of the product in float64, on x's device"""
    x, w, dy = x.double(), w.double(), dy.double()
    wm = w.transpose(1, 2) if transposed else w
    out, terms = [], [0] * w.shape[0]
    for f in (lambda t: t, torch.abs):
        if product == gp.FORWARD:
            r = x.new_zeros(x.shape[0], wm.shape[2])
        else:
            r = torch.zeros_like(x if product == gp.INPUT else wm)
        for g, (lo, hi) in enumerate(edges):
            m = g % w.shape[0]
            if product == gp.FORWARD:
                r[lo:hi] = f(x[lo:hi]) @ f(wm[m])
            elif product == gp.INPUT:
                r[lo:hi] = f(dy[lo:hi]) @ f(wm[m]).T
            else:
                r[m] += f(x[lo:hi]).T @ f(dy[lo:hi])
        out.append(r.transpose(1, 2) if transposed and product == gp.WEIGHT else r)
    for g, (lo, hi) in enumerate(edges):
        terms[g % w.shape[0]] += hi - lo
    return out[0].cpu(), out[1].cpu(), {gp.FORWARD: wm.shape[1], gp.INPUT: wm.shape[2], gp.WEIGHT: max(terms)}[product]


def run(dt, rows, K, N, groups, matrices, product, transposed):
    import mask_loss_amd
    ml = mask_loss_amd.mask_loss
    x, w, dy = (t.cuda() for t in base.make(rows, K, N, matrices, dt, transposed, rows + K))
    offsets = base.offsets_of(gp.counts_of(rows, groups), 1)
    o = torch.tensor(offsets).cuda()
    if product == gp.FORWARD:
        got = ml.grouped_matmul_forward(x, w, o, transposed)
    elif product == gp.INPUT:
        got = ml.grouped_matmul_backward_input(dy, w, o, transposed)
    else:
        got = ml.grouped_matmul_backward_weight(x, dy, o, matrices, transposed)
    base.check(got, *reference(x, w, dy, base.edges_of(offsets, rows), product, transposed), "product")


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("case", [i for i, c in enumerate(gp.CASES) if c[0] == gp.BF16])
def test_16_bit(dt, case):
    run(dt, *gp.CASES[case][4:])


@pytest.mark.parametrize("case", [i for i, c in enumerate(gp.CASES) if c[0] == gp.F32])
def test_float32(case):
    run("f32", *gp.CASES[case][4:])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_most_groups_on_the_largest_tile(dt):
    """4,000 matrices' weight gradients: the borders of the most groups beside the largest ring in LDS."""
    run(dt, 9000, 256, 256, 4000, 4000, gp.WEIGHT, False)
