"""Both gradients of a layer from one call, over operands of which one alone does not fit FP16 pairs: the form of a product is its own operands' affair,
so that each gradient is to the bit what it is when asked for by itself, and the input's gradient does not depend on the input."""
import numpy as np
import pytest
import torch

from test_gpu_fused_linear import E, down, fill, gt, near, randn, rel_of, up  # noqa: F401

pytestmark = pytest.mark.gpu


def spread(t, dim):
    """Sizes from 1 down to 2^-45 along a dimension: far more values below 2^-28 of the largest than are listed."""
    n = t.size(dim)
    shape = [1] * t.dim()
    shape[dim] = n
    return t * torch.exp2(-torch.linspace(0, 45, n, device="cuda").round()).reshape(shape)


KINDS = ["none", "x", "w", "g", "xw", "x inf", "w nan", "x strays"]


def operands(kind, x, w, g):
    if kind == "x" or kind == "xw":
        x = spread(x, 0)
    if kind == "w" or kind == "xw":
        w = spread(w, w.dim() - 2)
    if kind == "g":
        g = spread(g, 1)
    if kind == "x inf":
        x[7, 3] = float("inf")
    if kind == "w nan":
        w[..., 5, 9] = float("nan")
    if kind == "x strays":
        x[11] = 0
        x[11, 4] = 2.0 ** -40
    return x, w, g


def gradients(gt, m, x, g, counts, separate):  # noqa: F811
    m.gradWeight.fill(0.25)
    m.gradBias.zero()
    m.gradInput = gt.GPUTensor()
    inp, g = [up(gt, x), counts] if counts is not None else up(gt, x), up(gt, g)
    if separate:
        m.updateGradInput(inp, g)
        m.accGradParameters(inp, g, 0.5)
    else:
        m.backward(inp, g, 0.5)
    gi = m.gradInput if counts is None else m.gradInput[0]
    return down(gi).clone(), down(m.gradWeight).clone()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("counts,I,O", [(None, 2560, 2624), (None, 2531, 2602), ([6000, 0, 8200, 65, 1, 7400], 2560, 2624)])
def test_each_gradient_by_itself(gt, counts, I, O, kind):  # noqa: F811
    groups = [2600] if counts is None else counts
    R, n = sum(groups), len(groups)
    x, w, g = operands(kind, randn(1, R, I), randn(2, n, O, I) / I ** 0.5, randn(3, R, O))
    m = gt.nn.FusedLinear(I, O) if counts is None else gt.nn.GroupedLinear(n, I, O)
    fill(gt, m, w[0] if counts is None else w, torch.zeros(m.bias.shape, device="cuda"))
    before = gt.lib().THGPUProductCount(2)
    gi, gw = gradients(gt, m, x, g, counts, False)
    assert gt.lib().THGPUProductCount(2) - before == 2
    gi2, gw2 = gradients(gt, m, x, g, counts, True)
    if kind != "w nan":
        assert torch.equal(gi, gi2)
        # of another input the input's gradient is the same
        assert torch.equal(gi, gradients(gt, m, torch.ones_like(x), g, counts, False)[0])
    rows = torch.isfinite(x).all(1)
    assert torch.equal(gw.nan_to_num(), gw2.nan_to_num())
    # against the formulas, where these are finite
    X, G, W = torch.where(torch.isfinite(x), x, 0).double(), g.double(), torch.where(torch.isfinite(w), w, 0).double()
    ends = np.cumsum([0] + groups)
    columns = torch.isfinite(w).all(0).all(0)
    inputs = torch.isfinite(x).all(0)
    for e in range(n):
        p = slice(int(ends[e]), int(ends[e + 1]))
        near(gi[p][:, columns], (G[p] @ W[e])[:, columns], (rel_of(O) * (G[p].abs() @ W[e].abs()))[:, columns])
        want, size = G[p].t() @ X[p], G[p].abs().t() @ X[p].abs()
        keep = inputs if not rows[p].all() else torch.ones_like(inputs)
        near(gw[e][:, keep] if counts is not None else gw[:, keep], (0.25 + 0.5 * want)[:, keep], (0.5 * rel_of(groups[e]) * size + 2 * E * (0.25 + 0.5 * want.abs()))[:, keep])
