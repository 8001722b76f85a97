"""nn.LayerNorm against its formulas in 64 bits: lengths around every width the kernels have, unaligned and transposed inputs, rows that
are constant, far from zero, or hold an infinity or a NaN, and the sums of the weight's gradient."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24      # half a step of FP32


@pytest.fixture(scope="module")
def gt():
    import mcw_cppamp_torch_b200 as gt
    return gt


def randn(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, device="cuda", generator=g)


def up(gt, t):
    return gt.gpu(t.cpu().numpy())


def down(t):
    return torch.from_numpy(t.float()).cuda()


def chain(D):
    """Roundings that a term of a row's sum goes through: a thread of 256 or more adds up its share (a warp's lane at most 32 values), then the
    shuffles, the warps and the blocks of a cluster."""
    return D / 256 + 32 + 24


def check_forward(gt, m, x, w, b, eps=1e-5, input=None):
    got = down(m.forward(input if input is not None else up(gt, x))).reshape(x.shape)
    X, D = x.double(), x.size(-1)
    mean = X.mean(-1, keepdim=True)
    d = X - mean
    inv = (d.square().mean(-1, keepdim=True) + eps).rsqrt()
    u = d * inv
    want = u * w.double() + b.double()
    N = chain(D)
    # the mean is off by its rounding and by its correction's; each value less the mean once more; the variance by its chain (half of that in
    # inv), inv by a root and a division; the product and the sum once each
    off = E * (2 * mean.abs() + N * d.abs().mean(-1, keepdim=True)) * inv
    tol = w.double().abs() * (off + E * u.abs() * (N / 2 + 8)) + E * (2 * want.abs() + 2 * b.double().abs()) + 1e-37
    assert torch.all((got.double() - want).abs() <= tol)
    if m.train:
        assert torch.all((down(m.mean).double() - mean.squeeze(-1).reshape(-1)).abs() <= (E * (2 * mean.abs() + N * d.abs().mean(-1, keepdim=True))).reshape(-1))
        assert torch.all((down(m.invStd).double() / inv.reshape(-1) - 1).abs() <= E * (N / 2 + 8) + 4 * (off * off).reshape(-1))
    return got


def check_backward(gt, m, x, g, w, scale=1.0, x_in=None, g_in=None):
    """From the statistics that the forward pass has kept."""
    D, R = x.size(-1), x.numel() // x.size(-1)
    m.gradWeight.fill(0.5); m.gradBias.fill(-0.25)
    gi = down(m.backward(x_in if x_in is not None else up(gt, x), g_in if g_in is not None else up(gt, g), scale)).reshape(R, D)
    X, G, W = x.double().reshape(R, D), g.double().reshape(R, D), w.double()
    mean, inv = down(m.mean).double()[:, None], down(m.invStd).double()[:, None]
    u, gw = (X - mean) * inv, G * W
    a, c = gw.mean(1, keepdim=True), (gw * u).mean(1, keepdim=True)
    want = inv * (gw - a - u * c)
    N = chain(D)
    tol = inv * E * (4 * gw.abs() + (N + 4) * gw.abs().mean(1, keepdim=True) + u.abs() * (N + 8) * (gw * u).abs().mean(1, keepdim=True)) + 2 * E * want.abs()
    assert torch.all((gi.double() - want).abs() <= tol + 1e-37)
    # sums over the rows in any order: at most a rounding a row; u has three
    for got, start, terms in ((m.gradWeight, 0.5, G * u), (m.gradBias, -0.25, G)):
        want, mass = start + scale * terms.sum(0), abs(scale) * terms.abs().sum(0)
        assert torch.all((down(got).double() - want).abs() <= E * ((R + 6) * mass + 2 * want.abs() + 2 * abs(start)))
    return gi


def module(gt, *sizes, eps=1e-5, seed=3):
    m = gt.nn.LayerNorm(*sizes, eps=eps)
    w, b = 1 + 0.2 * randn(seed, m.size), 0.1 * randn(seed + 1, m.size)
    m.weight, m.bias = w.cpu().numpy(), b.cpu().numpy()
    return m.gpu(), w, b


SIZES = [1, 2, 3, 4, 7, 31, 32, 33, 64, 127, 128, 129, 333, 512, 1000, 1024, 1025, 1028, 2048, 2052, 4096, 4100, 5000, 8192, 8196, 10001, 16384, 16388,
         32768, 32772, 43264, 65536, 65540, 65537, 100003, 131072, 131076]


@pytest.mark.parametrize("rows,size", [(r, d) for r in (1, 3, 37, 301) for d in SIZES if r * d < 6e6])
def test_lengths(gt, rows, size):
    m, w, b = module(gt, size)
    x, g = 2 * randn(rows, rows, size) + 0.5, randn(rows + 1, rows, size)
    first = check_forward(gt, m, x, w, b)
    gi = check_backward(gt, m, x, g, w, scale=0.5)
    gw = down(m.gradWeight)
    assert torch.equal(check_forward(gt, m, x, w, b), first)                     # to the bit, also the sums over the rows
    assert torch.equal(check_backward(gt, m, x, g, w, scale=0.5), gi) and torch.equal(down(m.gradWeight), gw)


@pytest.mark.parametrize("rows,size", [(20001, 128), (5003, 1024), (4099, 2048), (2500, 333), (70001, 3)])
def test_many_rows(gt, rows, size):
    m, w, b = module(gt, size)
    x, g = randn(5, rows, size), randn(6, rows, size)
    check_forward(gt, m, x, w, b)
    check_backward(gt, m, x, g, w)


@pytest.mark.parametrize("size", [64, 4096, 20000])
def test_strides_and_addresses(gt, size):
    """Transposed inputs, rows at a pitch, rows and parameters that start off a 16-byte boundary."""
    rows = 29
    m, w, b = module(gt, size)
    x, g = randn(1, rows, size), randn(2, rows, size)
    wide = gt.GPUTensor(rows, size + 3).fill(7)
    views = [(up(gt, x.t().contiguous()).t(), up(gt, g.t().contiguous()).t()), (wide.narrow(2, 2, size), up(gt, g))]
    flat = gt.GPUTensor(rows * size + 1).narrow(1, 2, rows * size).view(rows, size)
    views.append((flat, flat.clone()))
    for i, (xv, gv) in enumerate(views):
        if i:
            xv.copy(x.cpu().numpy())
        if i == 2:
            gv = gt.GPUTensor(rows * size + 3).narrow(1, 4, rows * size).view(rows, size).copy(g.cpu().numpy())
        check_forward(gt, m, x, w, b, input=xv)
        check_backward(gt, m, x, g, w, x_in=xv, g_in=gv)
    keep = gt.GPUTensor(4 * size + 4)
    for i, name in enumerate(("weight", "bias", "gradWeight", "gradBias")):
        setattr(m, name, keep.narrow(1, 2 + i * size, size).copy(getattr(m, name)))
    check_forward(gt, m, x, w, b)
    check_backward(gt, m, x, g, w)


def test_more_dimensions(gt):
    m, w, b = module(gt, 6, 5, 7)
    x, g = randn(1, 4, 3, 6, 5, 7), randn(2, 4, 3, 6, 5, 7)
    m.forward(up(gt, x))
    assert m.output.size() == (4, 3, 6, 5, 7) and m.mean.size() == (12,)
    check_forward(gt, m, x.reshape(12, 210), w, b)
    check_backward(gt, m, x.reshape(12, 210), g.reshape(12, 210), w)
    m.forward(up(gt, x[0, 0]))
    assert m.output.size() == (6, 5, 7) and m.mean.size() == (1,)


@pytest.mark.parametrize("size", [5, 100, 1024, 3000, 16384, 50000, 140000])
def test_rows_that_are_alike_or_far_away(gt, size):
    """Constant rows come to the bias; rows far from zero keep their spread; tiny and huge ones their direction."""
    m, w, b = module(gt, size)
    x = randn(1, 9, size)
    x[0], x[1] = 3.25, 0
    x[2] = x[2] + 4096.0
    x[3] = (x[3] * 64).round() / 64 + 1e4
    x[4], x[5] = x[4] * 1e-12, x[5] * 1e15
    check_forward(gt, m, x, w, b)
    out = down(m.output)
    assert torch.equal(out[0], b) and torch.equal(out[1], b)
    check_backward(gt, m, x, randn(2, 9, size), w)


@pytest.mark.parametrize("size", [8, 1000, 4096, 40000, 140000])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_a_row_with_no_statistics_spoils_itself_alone(gt, size, value):
    m, w, b = module(gt, size)
    x, g = randn(1, 40, size), randn(2, 40, size)
    clean = x.clone()
    want = check_forward(gt, m, clean, w, b)
    gi = down(m.backward(up(gt, clean), up(gt, g)))
    x[17, size // 2] = value
    got = down(m.forward(up(gt, x)))
    keep = torch.arange(40, device="cuda") != 17
    assert torch.equal(got[keep], want[keep]) and got[17].isnan().all()
    back = down(m.backward(up(gt, x), up(gt, g)))
    assert torch.equal(back[keep], gi[keep]) and back[17].isnan().all()
    assert down(m.gradWeight).isnan().all() and not down(m.gradBias).isnan().any()


def test_parts_of_a_backward_pass(gt):
    """updateGradInput and accGradParameters give what backward gives; no parameters, no statistics kept, no gradInput, in a container."""
    x, g = randn(1, 65, 700), randn(2, 65, 700)
    m, w, b = module(gt, 700)
    check_forward(gt, m, x, w, b)
    m.zeroGradParameters()
    both = [down(t).clone() for t in (m.backward(up(gt, x), up(gt, g), 2.0), m.gradWeight, m.gradBias)]
    m.zeroGradParameters()
    m.gradInput = gt.GPUTensor()
    one = down(m.updateGradInput(up(gt, x), up(gt, g)))
    m.accGradParameters(up(gt, x), up(gt, g), 2.0)
    for a, c in zip(both, (one, down(m.gradWeight), down(m.gradBias))):
        assert torch.equal(a, c)
    m.gradInput = None
    m.zeroGradParameters()
    assert m.backward(up(gt, x), up(gt, g), 2.0) is None and torch.equal(down(m.gradWeight), both[1])
    plain = gt.nn.LayerNorm(700, affine=False).gpu()
    ones, zeros = torch.ones(700, device="cuda"), torch.zeros(700, device="cuda")
    check_forward(gt, plain, x, ones, zeros)
    same, _, _ = module(gt, 700)
    same.weight.fill(1)
    same.forward(up(gt, x))
    assert torch.equal(down(plain.backward(up(gt, x), up(gt, g))), down(same.backward(up(gt, x), up(gt, g))))
    plain.accGradParameters(up(gt, x), up(gt, g))
    m.evaluate()
    kept = down(m.mean).clone()
    check_forward(gt, m, x + 1, w, b)
    assert torch.equal(down(m.mean), kept)
    m.training()
    assert m.train
    net = gt.nn.Sequential().add(m).add(gt.nn.ReLU())
    assert net.evaluate() is net and not m.train


def test_empty_batches(gt):
    m, _, _ = module(gt, 12)
    empty = gt.GPUTensor()
    m.gradWeight.fill(3)
    assert m.forward(empty).nElement() == 0 and m.backward(empty, gt.GPUTensor()).nElement() == 0
    assert torch.all(down(m.gradWeight) == 3)


def test_differences(gt):
    """The gradients against differences of the loss sum(g * y) in 64 bits of the module's own outputs."""
    m, w, b = module(gt, 24)
    x, g = randn(1, 5, 24), randn(2, 5, 24)
    m.forward(up(gt, x))
    m.zeroGradParameters()
    gi = down(m.backward(up(gt, x), up(gt, g))).double()
    h = 2.0 ** -8

    def loss(xv):
        return (down(m.forward(up(gt, xv))).double() * g.double()).sum()
    for i, j in ((0, 0), (2, 7), (4, 23)):
        d = torch.zeros_like(x)
        d[i, j] = h
        hi, lo = x + d, x - d
        slope = (loss(hi) - loss(lo)) / (hi[i, j].double() - lo[i, j].double())
        # the outputs' roundings over 2h, and h^2 / 6 times a third derivative of a few tens
        assert abs(slope - gi[i, j]) <= 24 * 8 * E * 10 / (2 * h) + h * h * 10
