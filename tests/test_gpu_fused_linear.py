"""nn.FusedLinear and nn.GroupedLinear against their formulas in 64 bits: every way a product is computed (rows of one to thousands, sizes that
no tile or 16-byte access divides), activations, residuals, strides, groups of all sizes with empty ones among them, gradients."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
REL = 2.0 ** -19     # of the sum of |products|: the dropped terms and truncating chains of 3xTF32, which FP16 pairs stay below
ACTS = ["none", "relu", "gelu", "silu"]


@pytest.fixture(scope="module")
def gt():
    import mcw_cppamp_torch_b200 as gt
    gt.set_math_mode("fp32x3")
    return gt


def randn(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, device="cuda", generator=g)


def up(gt, t):
    return gt.gpu(t.cpu().numpy())


def down(t):
    return torch.from_numpy(t.float()).cuda()


def act(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return z * 0.5 * torch.erfc(-z * math.sqrt(0.5))
    return z * torch.sigmoid(z) if name == "silu" else z


def slope(z, name):
    if name == "relu":
        return (z > 0).double()
    if name == "gelu":
        return 0.5 * torch.erfc(-z * math.sqrt(0.5)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "silu":
        s = torch.sigmoid(z)
        return s + z * s * (1 - s)
    return torch.ones_like(z)


def rel_of(terms, mode="fp32x3"):
    """Error of a product's sum, of the sum of |products|: one rounding for each 32 terms; simt at most one a term; bf16 operands 2^-8 each."""
    return {"fp32x3": REL, "simt": terms * E, "bf16": 2.0 ** -7}[mode] + (terms / 32 + 34) * E


def near(got, want, tol):
    assert got.shape == want.shape
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), float((got.double() - want).abs().max()), float(tol.min()))


def y_tolerance(z, zt, y, name, r=None):
    # |act'| <= 1.13; erfc, exp and the division are within a few steps of their values: 8 half steps each of what they make
    t = 1.13 * zt + 16 * E * y.abs() + 2 * E * z.abs() * (name != "none")
    return t if r is None else t + E * (y.abs() + r.abs())


def fill(gt, m, w, b):
    m.weight, m.bias = w.cpu().numpy(), b.cpu().numpy()
    return m.gpu()


def check_linear(gt, R, I, O, name, residual=False, mode="fp32x3", views=lambda gt, t: up(gt, t), scale=0.5, backward=True):
    x, w, b, r, g = randn(1, R, I), randn(2, O, I) / I ** 0.5, 0.1 * randn(3, O), randn(4, R, O), randn(5, R, O)
    m = fill(gt, gt.nn.FusedLinear(I, O, name), w, b)
    X, W, B, G = x.double(), w.double(), b.double(), g.double()
    z = X @ W.t() + B
    zt = rel_of(I, mode) * (X.abs() @ W.abs().t() + B.abs())
    if mode == "bf16":
        zt = zt + 1e-30
    y = act(z, name)
    xin = views(gt, x)
    inp = [xin, views(gt, r)] if residual else xin
    tol = y_tolerance(z, zt, y, name, r.double() if residual else None)
    near(down(m.forward(inp)), y + r.double() if residual else y, tol)
    train = down(m.output)
    if name != "none":
        near(down(m.preactivation), z, zt)
    m.evaluate()
    m.output = gt.GPUTensor()
    assert torch.equal(down(m.forward(inp)), train)
    m.training()
    if not backward:
        return
    m.forward(inp)
    # the backward pass goes by what the forward pass has kept
    zk = down(m.preactivation).double() if name != "none" else z
    s = slope(zk, name)
    gz = G * s
    # the slopes of gelu and silu are sums of two terms below 1 + |z|
    gzt = (16 * E * G.abs() * (1 + zk.abs().clamp(max=8)) if name in ("gelu", "silu") else torch.zeros_like(G)) + E * gz.abs()
    if mode == "bf16":
        gzt = gzt + 2.0 ** -8 * gz.abs()
    m.gradWeight.fill(0.25); m.gradBias.fill(-0.5)
    gi = m.backward(inp, views(gt, g), scale)
    if residual:
        assert len(gi) == 2 and torch.equal(down(gi[1]), g)
        gi = gi[0]
    near(down(gi), gz @ W, rel_of(O, mode) * (gz.abs() @ W.abs()) + gzt @ W.abs())
    near(down(m.gradWeight), 0.25 + scale * (gz.t() @ X),
         scale * (rel_of(R, mode) * (gz.abs().t() @ X.abs()) + gzt.t() @ X.abs()) + 2 * E * (0.25 + scale * (gz.t() @ X).abs()))
    near(down(m.gradBias), -0.5 + scale * gz.sum(0), scale * ((R + 4) * E * gz.abs().sum(0) + gzt.sum(0)) + 2 * E)
    # the two parts by themselves
    first = [down(t).clone() for t in (gi, m.gradWeight, m.gradBias)]
    m.gradInput = gt.GPUTensor()
    m.gradWeight.fill(0.25); m.gradBias.fill(-0.5)
    gi = m.updateGradInput(inp, views(gt, g))
    m.accGradParameters(inp, views(gt, g), scale)
    for a, c in zip(first, (gi[0] if residual else gi, m.gradWeight, m.gradBias)):
        assert torch.equal(a, down(c))


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("R,I,O", [(1, 1, 1), (1, 9216, 400), (2, 512, 512), (3, 64, 1000), (5, 333, 77), (8, 1024, 600), (9, 40, 8), (17, 100, 333),
                                   (64, 256, 256), (100, 1000, 130), (129, 65, 257), (300, 512, 1000), (777, 1531, 1001), (513, 2048, 1024)])
def test_sizes(gt, R, I, O, name):
    check_linear(gt, R, I, O, name, residual=(R + O) % 2 == 0)


@pytest.mark.parametrize("R,I,O,name", [(2048, 2048, 2304, "gelu"), (2500, 2222, 2600, "silu"), (4100, 1030, 4100, "relu"), (256, 4096, 4096, "gelu"),
                                        (4097, 2050, 2304, "none"), (8192, 512, 260, "silu"), (40, 4100, 4096, "gelu")])
@pytest.mark.parametrize("residual", [False, True])
def test_large(gt, R, I, O, name, residual):
    """Products over FP16 pairs and FP32 values on the two-SM engine, whole tiles and cut ones."""
    check_linear(gt, R, I, O, name, residual)


@pytest.mark.parametrize("mode", ["simt", "bf16"])
@pytest.mark.parametrize("R,I,O", [(1, 128, 64), (33, 200, 140), (300, 512, 300), (2048, 1024, 1024)])
def test_math_modes(gt, mode, R, I, O):
    gt.set_math_mode(mode)
    try:
        for name in ("gelu", "none"):
            check_linear(gt, R, I, O, name, residual=True, mode=mode)
    finally:
        gt.set_math_mode("fp32x3")


@pytest.mark.parametrize("R", [1, 6, 70, 700])
def test_strides(gt, R):
    """Rows at a pitch, off 16 bytes, and transposed."""
    def pitched(gt, t):
        return gt.GPUTensor(t.size(0), t.size(1) + 5).fill(float("nan")).narrow(2, 3, t.size(1)).copy(t.cpu().numpy())

    def transposed(gt, t):
        return up(gt, t.t().contiguous()).t()
    for views in (pitched, transposed):
        check_linear(gt, R, 260, 132, "gelu", residual=True, views=views)
        check_linear(gt, R, 260, 132, "none", residual=False, views=views)


@pytest.mark.parametrize("R,I,O", [(3000, 2304, 2304), (2304, 2560, 3000)])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("train", [True, False])
def test_values_that_pairs_do_not_hold(gt, R, I, O, residual, train):
    """A few values far below the largest of their operand are added to the products on their own: the activation is of the whole sum."""
    x, w = randn(1, R, I), randn(2, O, I)
    x[:, 0] = 0
    x[5], w[7] = 0, 0
    x[5, 0], w[7, 3] = 2.0 ** -40, 2.0 ** -41          # all there is in their row
    x[9, 9] = 2.0 ** -45
    x[11, 3] = 2.0 ** 20
    b, r = torch.zeros(O, device="cuda"), randn(4, R, O)
    for name in ("silu", "relu", "gelu"):
        m = fill(gt, gt.nn.FusedLinear(I, O, name), w, b)
        m.train = train
        inp = [up(gt, x), up(gt, r)] if residual else up(gt, x)
        got = down(m.forward(inp))
        X, W = x.double(), w.double()
        z = X @ W.t()
        zt = rel_of(I) * (X.abs() @ W.abs().t())
        y = act(z, name)
        # next to zero the activation's slope is its value over z: tiny sums keep their leading bits
        near(got, y + r.double() if residual else y, y_tolerance(z, zt, y, name, r.double() if residual else None))
        if train:
            near(down(m.preactivation), z, zt)


def test_far_arguments(gt):
    """Activations where exponentials end: large, tiny, infinite and not-a-number sums."""
    z = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 0.5, -0.5, 4, -4, 9, -9, 13, -13, 20, -20, 88, -88, 104, -104, 1e4, -1e4, 3e38, -3e38, float("inf"),
                      float("nan")], device="cuda")
    n = z.numel()
    one, zero = torch.ones(1, 1, device="cuda"), torch.zeros(n, device="cuda")
    for name in ACTS:
        m = fill(gt, gt.nn.FusedLinear(1, n, name), torch.ones(n, 1, device="cuda"), zero)
        m.bias.copy(z.cpu().numpy())
        m.weight.zero()
        got = down(m.forward(up(gt, one)))[0]
        want = act(z.double(), name)
        if name == "relu":
            want = torch.where(z > 0, z, torch.zeros_like(z)).double()      # a NaN gives zero, as nn.Threshold's does
        num = ~want.isnan()
        assert torch.equal(got.isnan(), ~num)
        fin = num & want.isfinite()
        assert torch.equal(got[num & ~fin].double(), want[num & ~fin])
        # erfc's argument z / sqrt 2 is off by two half steps (the constant's, the product's), and erfc(a) falls as exp(-a^2): a relative
        # 2 a^2 = z^2 times that
        argument = 2 * z[fin].double().square() if name == "gelu" else 0
        assert torch.all((got[fin].double() - want[fin]).abs() <= (16 + argument) * E * want[fin].abs() + 1e-37)
        g = down(m.updateGradInput(up(gt, one), up(gt, torch.ones(1, n, device="cuda"))))
        if name != "none":
            back = down(m.gradPreactivation)[0]
            ws = torch.where(z > 0, 1.0, 0.0).double() if name == "relu" else slope(z.double(), name)
            fin = ws.isfinite()
            assert torch.all((back[fin].double() - ws[fin]).abs() <= 24 * E * (1 + z[fin].double().abs().nan_to_num().clamp(max=8)) + 1e-37)
        assert g.numel() == 1


def test_empty_and_containers(gt):
    m = gt.nn.FusedLinear(6, 4, "gelu").gpu()
    empty = gt.GPUTensor()
    m.gradWeight.fill(2)
    assert m.forward(empty).nElement() == 0 and m.backward(empty, gt.GPUTensor()).nElement() == 0
    assert m.forward([empty, gt.GPUTensor()]).nElement() == 0
    assert torch.all(down(m.gradWeight) == 2)
    q = gt.nn.GroupedLinear(3, 6, 4, "silu").gpu()
    q.gradWeight.fill(2)
    assert q.forward([empty, [0, 0, 0]]).nElement() == 0 and q.backward([empty, [0, 0, 0]], gt.GPUTensor())[0].nElement() == 0
    assert torch.all(down(q.gradWeight) == 2)
    net = gt.nn.Sequential().add(gt.nn.FusedLinear(6, 5, "relu")).add(gt.nn.FusedLinear(5, 3)).add(gt.nn.LogSoftMax()).gpu()
    x, g = randn(1, 7, 6), randn(2, 7, 3)
    out = down(net.forward(up(gt, x))).clone()
    same = gt.nn.Sequential().add(gt.nn.Linear(6, 5)).add(gt.nn.ReLU()).add(gt.nn.Linear(5, 3)).add(gt.nn.LogSoftMax()).gpu()
    for a, c in ((0, 0), (1, 2)):
        same.modules[c].weight.copy(net.modules[a].weight); same.modules[c].bias.copy(net.modules[a].bias)
    near(out, down(same.forward(up(gt, x))).double(), torch.full_like(out, 1e-5).double())
    near(down(net.backward(up(gt, x), up(gt, g))), down(same.backward(up(gt, x), up(gt, g))).double(), torch.full((7, 6), 1e-4, device="cuda").double())


# ------------------------------------------------------------------ groups
def check_groups(gt, counts, I, O, name, scale=0.5, views=lambda gt, t: up(gt, t), pad=0, backward=True, mode="fp32x3"):
    T, n = int(sum(counts)), len(counts)
    x, w, b, g = randn(1, T, I), randn(2, n, O, I) / I ** 0.5, 0.1 * randn(3, n, O), randn(4, T, O)
    m = fill(gt, gt.nn.GroupedLinear(n, I, O, name), w, b)
    X, W, B, G = x.double(), w.double(), b.double(), g.double()
    ends = np.cumsum([0] + [int(c) for c in counts])
    at = [slice(int(a), int(c)) for a, c in zip(ends[:-1], ends[1:])]
    z = torch.cat([X[p] @ W[e].t() + B[e] for e, p in enumerate(at)])
    zt = torch.cat([rel_of(I, mode) * (X[p].abs() @ W[e].abs().t() + B[e].abs()) for e, p in enumerate(at)])
    y = act(z, name)
    xin = views(gt, x)
    near(down(m.forward([xin, counts])), y, y_tolerance(z, zt, y, name))
    if name != "none":
        near(down(m.preactivation), z, zt)
    train = down(m.output)
    m.evaluate()
    m.output = gt.GPUTensor()
    assert torch.equal(down(m.forward([xin, counts])), train)
    m.training()
    if not backward:
        return
    m.forward([xin, counts])
    zk = down(m.preactivation).double() if name != "none" else z
    gz = G * slope(zk, name)
    gzt = (16 * E * G.abs() * (1 + zk.abs().clamp(max=8)) if name in ("gelu", "silu") else torch.zeros_like(G)) + E * gz.abs()
    m.gradWeight.fill(0.25); m.gradBias.fill(-0.5)
    gi, none = m.backward([xin, counts], views(gt, g), scale)
    assert none is None
    near(down(gi), torch.cat([gz[p] @ W[e] for e, p in enumerate(at)]),
         torch.cat([rel_of(O, mode) * (gz[p].abs() @ W[e].abs()) + gzt[p] @ W[e].abs() for e, p in enumerate(at)]))
    gw, gb = down(m.gradWeight), down(m.gradBias)
    for e, p in enumerate(at):
        want = scale * (gz[p].t() @ X[p])
        near(gw[e], 0.25 + want, scale * (rel_of(counts[e], mode) * (gz[p].abs().t() @ X[p].abs()) + gzt[p].t() @ X[p].abs()) + 2 * E * (0.25 + want.abs()))
        near(gb[e], -0.5 + scale * gz[p].sum(0), scale * ((counts[e] + 4) * E * gz[p].abs().sum(0) + gzt[p].sum(0)) + 2 * E)
        if counts[e] == 0:
            assert torch.all(gw[e] == 0.25) and torch.all(gb[e] == -0.5)
    first = [down(t).clone() for t in (gi, m.gradWeight, m.gradBias)]
    m.gradInput = gt.GPUTensor()
    m.gradWeight.fill(0.25); m.gradBias.fill(-0.5)
    gi = m.updateGradInput([xin, counts], views(gt, g))[0]
    m.accGradParameters([xin, counts], views(gt, g), scale)
    for a, c in zip(first, (gi, m.gradWeight, m.gradBias)):
        assert torch.equal(a, down(c))


COUNTS = {
    "one": [1], "one of many": [0, 0, 1, 0, 0, 0], "last": [0, 0, 7], "few": [1, 0, 2, 0, 0, 1, 3, 0], "edges": [63, 64, 65, 0, 128, 127, 129, 1],
    "mixed": [300, 1, 0, 77, 512, 31, 33, 2], "even": [96] * 8, "single": [700], "many": [3, 0, 1] * 50,
}


@pytest.mark.parametrize("I,O", [(64, 96), (33, 17), (256, 260), (100, 1), (1, 40), (515, 333)])
@pytest.mark.parametrize("which", list(COUNTS))
def test_groups(gt, which, I, O):
    check_groups(gt, COUNTS[which], I, O, ACTS[(I + len(which)) % 4])


@pytest.mark.parametrize("counts,I,O,name", [([900, 30, 2200, 0, 511, 1, 257, 256], 1024, 1408, "silu"), ([4000, 96], 512, 2048, "gelu"),
                                             ([5, 0, 9, 1, 0, 3, 2, 4] * 8, 1024, 1024, "relu"), ([2048, 2048], 2048, 2048, "none")])
def test_large_groups(gt, counts, I, O, name):
    check_groups(gt, counts, I, O, name)


@pytest.mark.parametrize("mode", ["simt", "bf16"])
def test_groups_in_other_modes(gt, mode):
    gt.set_math_mode(mode)
    try:
        check_groups(gt, [200, 0, 3, 150], 128, 96, "gelu", mode="simt" if mode == "simt" else "bf16")
    finally:
        gt.set_math_mode("fp32x3")


def test_group_strides(gt):
    def pitched(gt, t):
        return gt.GPUTensor(t.size(0), t.size(1) + 3).fill(float("nan")).narrow(2, 2, t.size(1)).copy(t.cpu().numpy())

    def transposed(gt, t):
        return up(gt, t.t().contiguous()).t()
    for views in (pitched, transposed):
        check_groups(gt, [40, 0, 3, 150], 128, 96, "gelu", views=views)
        check_groups(gt, [40, 0, 3, 150], 128, 96, "none", views=views)


@pytest.mark.parametrize("I,O", [(96, 64), (130, 70)])
def test_a_group_keeps_to_itself(gt, I, O):
    """Rows and weights that are infinite or NaN reach their own group's results alone, whatever the counts."""
    counts = [70, 5, 0, 130, 64, 1, 30]
    T, n = sum(counts), len(counts)
    x, w, b, g = randn(1, T, I), randn(2, n, O, I), randn(3, n, O), randn(4, T, O)
    out = []
    for bad in (False, True):
        if bad:
            x[70:75], w[3], g[269:270] = float("nan"), float("inf"), float("nan")
        m = fill(gt, gt.nn.GroupedLinear(n, I, O, "none"), w, b)
        m.zeroGradParameters()
        y = down(m.forward([up(gt, x), counts]))
        gi = down(m.backward([up(gt, x), counts], up(gt, g))[0])
        out.append((y, gi, down(m.gradWeight), down(m.gradBias)))
    rows = torch.ones(T, dtype=torch.bool, device="cuda")
    rows[70:205], rows[269] = False, False
    groups = torch.tensor([e not in (1, 3, 5) for e in range(n)], device="cuda")
    for a, c in zip(*out):
        keep = rows if a.size(0) == T else groups
        assert torch.equal(a[keep], c[keep]) and torch.isfinite(c[keep]).all()


@pytest.mark.parametrize("kind", ["plain", "strays", "wide", "odd"])
@pytest.mark.parametrize("name", ["gelu", "none"])
@pytest.mark.parametrize("large", [False, True])
def test_groups_over_pairs(gt, kind, name, large):
    """Products whose operands are split into FP16 halves: padded groups, values that halves do not hold (a few: added on their own; many: the same
    launch multiplies FP32 values), in all three passes."""
    counts, I, O = [1500, 0, 2300, 65, 1, 2230], 1536, 1600
    if kind == "odd":
        I, O = 1531, 1601
    if large:                                                    # (at the sizes above the engine takes the FP32 values)
        counts, I, O = [6000, 0, 8200, 65, 1, 7400], I + 1024, O + 1024
    T, n = sum(counts), len(counts)
    x, w, b, g = randn(1, T, I), randn(2, n, O, I) / I ** 0.5, 0.1 * randn(3, n, O), randn(4, T, O)
    b[:, 3] = 0
    if kind == "strays":
        for r in (0, 1499, 1500, 3799, 3864, 3865, T - 1):       # rows with one value each, far below the largest
            x[r] = 0
            x[r, r % I] = 2.0 ** -38
            g[r] = 0
            g[r, r % O] = 2.0 ** -37
        w[2, 3] = 0
        w[2, 3, 7] = 2.0 ** -40                                  # a line of a weight
        w[5, :, 11] = 0
        w[5, 9, 11] = 2.0 ** -41                                 # a column of another
        w[1, 0, 0] = 2.0 ** -42                                  # of a group without rows
    if kind == "wide":
        x = x * torch.exp2(-torch.linspace(0, 45, T, device="cuda").round())[:, None]
        w = w * torch.exp2(-torch.linspace(0, 40, O, device="cuda").round())[None, :, None]
    m = fill(gt, gt.nn.GroupedLinear(n, I, O, name), w, b)
    X, W, B, G = x.double(), w.double(), b.double(), g.double()
    ends = np.cumsum([0] + counts)
    at = [slice(int(a), int(c)) for a, c in zip(ends[:-1], ends[1:])]
    L = gt.lib()
    before = L.THGPUProductCount(2)
    m.forward([up(gt, x), counts])
    z = torch.cat([X[p] @ W[e].t() + B[e] for e, p in enumerate(at)])
    zt = torch.cat([rel_of(I) * (X[p].abs() @ W[e].abs().t() + B[e].abs()) for e, p in enumerate(at)])
    y = act(z, name)
    near(down(m.output), y, y_tolerance(z, zt, y, name))
    if name != "none":
        near(down(m.preactivation), z, zt)
        m.preactivation.fill(30)                                 # slopes of one: the gradients' rows keep their sizes
    m.gradWeight.zero(); m.gradBias.zero()
    gi = down(m.backward([up(gt, x), counts], up(gt, g), 1.0)[0])
    if large:                                                    # (of odd sizes the passes go value by value, which suits pairs less)
        assert L.THGPUProductCount(2) - before >= (1 if kind == "odd" else 3)
    near(gi, torch.cat([G[p] @ W[e] for e, p in enumerate(at)]), torch.cat([(rel_of(O) + 8 * E) * (G[p].abs() @ W[e].abs()) for e, p in enumerate(at)]))
    gw = down(m.gradWeight)
    for e, p in enumerate(at):
        near(gw[e], G[p].t() @ X[p], (rel_of(counts[e]) + 8 * E) * (G[p].abs().t() @ X[p].abs()))
    first = [t.clone() for t in (gi, gw)]
    m.gradInput = gt.GPUTensor()
    m.gradWeight.zero()
    assert torch.equal(down(m.updateGradInput([up(gt, x), counts], up(gt, g))[0]), first[0])
    m.accGradParameters([up(gt, x), counts], up(gt, g), 1.0)
    assert torch.equal(down(m.gradWeight), first[1])


def test_groups_with_infinite_rows_over_pairs(gt):
    """An infinity makes the operands stay in FP32; its row's and its group's results are its own."""
    counts, I, O = [2000, 2100, 1900], 1536, 1536
    T = sum(counts)
    x, w, b, g = randn(1, T, I), randn(2, 3, O, I) / I ** 0.5, randn(3, 3, O), randn(4, T, O)
    m = fill(gt, gt.nn.GroupedLinear(3, I, O, "none"), w, b)
    x[2500, 7] = float("inf")
    y = down(m.forward([up(gt, x), counts]))
    m.gradWeight.zero()
    m.backward([up(gt, x), counts], up(gt, g))
    rows = torch.arange(T, device="cuda") != 2500
    X, W = x.double(), w.double()
    for e, p in enumerate((slice(0, 2000), slice(2000, 4100), slice(4100, 6000))):
        k = rows[p]
        near(y[p][k], (X[p] @ W[e].t() + b[e].double())[k], (rel_of(I) * (X[p].abs() @ W[e].abs().t() + b[e].abs().double()))[k])
        if e != 1:
            near(down(m.gradWeight)[e], g[p].double().t() @ X[p], (rel_of(counts[e]) + 4 * E) * (g[p].abs().double().t() @ X[p].abs()))


@pytest.mark.parametrize("last", [0, 1, 16, 40])
@pytest.mark.parametrize("n,I,O", [(20000, 8, 8), (70000, 3, 5), (3000, 64, 32), (2, 1, 4200000)])
def test_many_groups_and_many_columns(gt, n, I, O, last):
    """More groups, or more columns, than a launch has of blocks to count them by; `last`: rows of the last group, few or not (an empty tensor has no
    dimensions)."""
    counts = np.arange(n) % 3
    counts[-1] = last
    e = torch.from_numpy(np.repeat(np.arange(n), counts)).cuda()
    T = len(e)
    x, w, b, g = randn(1, T, I), randn(2, n, O, I) / I ** 0.5, 0.1 * randn(3, n, O), randn(4, T, O)
    m = fill(gt, gt.nn.GroupedLinear(n, I, O), w, b)
    X, W, B, G = x.double(), w.double()[e], b.double()[e], g.double()
    near(down(m.forward([up(gt, x), counts])).reshape(T, O), torch.einsum("ti,toi->to", X, W) + B, rel_of(I) * (torch.einsum("ti,toi->to", X.abs(), W.abs()) + B.abs()))
    m.gradWeight.fill(0.25); m.gradBias.fill(-0.5)
    gi = m.backward([up(gt, x), counts], up(gt, g), 0.5)[0]
    near(down(gi).reshape(T, I), torch.einsum("to,toi->ti", G, W), rel_of(O) * torch.einsum("to,toi->ti", G.abs(), W.abs()))
    for k, (got, start, terms) in enumerate(((down(m.gradWeight), 0.25, G[:, :, None] * X[:, None, :]), (down(m.gradBias), -0.5, G))):
        sums = torch.zeros(got.shape, dtype=torch.float64, device="cuda")
        want, size = sums.index_add(0, e, terms), sums.index_add(0, e, terms.abs())
        near(got, start + 0.5 * want, 0.5 * rel_of(2) * size + 2 * E * (abs(start) + 0.5 * want.abs()))


@pytest.mark.parametrize("R", [1, 2, 4, 7, 15, 16, 17])
@pytest.mark.parametrize("I,O", [(1, 1), (4, 9), (130, 64), (333, 515), (1024, 70), (1100, 33), (5000, 3)])
def test_weight_gradients_of_few_rows(gt, R, I, O):
    """Rows of all strides, pitches that 16-byte accesses take and others, columns of one block and of several, empty groups around."""
    def wide(gt, t):
        return up(gt, torch.cat([t, t.flip(0)], 1)).narrow(2, 1, t.shape[1])

    for views in (lambda gt, t: up(gt, t), wide, lambda gt, t: up(gt, t.t().contiguous()).t()):
        check_linear(gt, R, I, O, "none", views=views)
        check_groups(gt, [0, R, 1, 0, 2, R], I, O, "none", views=views)


@pytest.mark.parametrize("counts", [[1] * 8, [2, 0, 1, 2] * 3, [4, 3, 0, 1, 2] * 2, [1] * 40 + [0] * 5 + [4], [8, 1, 7, 5] * 2, [9] + [1] * 9, [3] * 7])
@pytest.mark.parametrize("I,O", [(1, 1), (130, 64), (128, 513), (333, 515), (260, 2049), (5000, 70)])
def test_input_gradients_of_few_rows(gt, counts, I, O):
    """Rows of weights that a block's pieces divide and others, one piece of them and several, columns of one tile and of several."""
    check_groups(gt, counts, I, O, "silu")
