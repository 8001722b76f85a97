"""optim.AdamW against its definition: in 32 bits within the roundings of each step, in 8 bits code for code against the same FP32 operations in numpy."""
import ctypes
import io
import pickle

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F = np.float32
SIZES = [(1,), (255,), (256,), (257,), (3, 7), (2048,), (2049,), (64, 100), (5000,), (1, 1)]


@pytest.fixture(scope="module")
def gt():
    import mcw_cppamp_torch_b200 as gt
    return gt


def normal(seed, *shape):
    return np.random.RandomState(seed).standard_normal(shape).astype(F)


def views(gt, arrays, off=0):
    """Tensors side by side in one storage, as getParameters leaves them, the first `off` values in."""
    flat = gt.GPUTensor(off + sum(a.size for a in arrays)).fill(0.0)
    out, at = [], off + 1
    for a in arrays:
        v = flat.narrow(1, at, a.size).view(*a.shape)
        v.copy(a)
        out.append(v)
        at += a.size
    return out


def one_step(w, g, m, v, t, lr, b1, b2, eps, decay):
    """In 64 bits, from FP32 states."""
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    return w * (1 - lr * decay) - lr / (1 - b1 ** t) * m / (np.sqrt(v / (1 - b2 ** t)) + eps), m, v


@pytest.mark.parametrize("lr,b1,b2,eps,decay", [(1e-3, 0.9, 0.999, 1e-8, 0.01), (0.1, 0.0, 0.5, 1e-3, 0.0), (3e-4, 0.95, 0.9999, 1e-6, 0.1), (0.0, 0.9, 0.99, 1e-8, 1.0)])
@pytest.mark.parametrize("off", [0, 1, 4])
def test_steps_in_32_bits(gt, lr, b1, b2, eps, decay, off):
    w, g = [normal(i, *s) for i, s in enumerate(SIZES)], [normal(50 + i, *s) for i, s in enumerate(SIZES)]
    W, G = views(gt, w, off), views(gt, g, off)
    opt = gt.optim.AdamW(W, G, learningRate=lr, beta1=b1, beta2=b2, epsilon=eps, weightDecay=decay)
    if off == 4:
        opt.mean, opt.square = views(gt, [np.zeros(s, F) for s in SIZES], 4), views(gt, [np.zeros(s, F) for s in SIZES], 4)
    m, v = ([np.zeros(s, F) for s in SIZES] for _ in range(2))
    for t in range(1, 5):
        for i in range(len(SIZES)):
            G[i].copy(np.float32(10.0 ** (t - 3)) * g[i])
        opt.update()
        assert opt.step.float().tolist() == [t, 0]
        for i in range(len(SIZES)):
            gi = np.float32(10.0 ** (t - 3)) * g[i]
            a = [x.astype(np.float64) for x in (w[i], gi, m[i], v[i])]
            ww, mm, vv = one_step(*a, t, lr, b1, b2, eps, decay)
            m[i], v[i], old, w[i] = opt.mean[i].float(), opt.square[i].float(), w[i], W[i].float()
            # constants rounded to FP32 (half a step), products and sums of two terms; a factor 1 - beta loses what beta's half step is of it
            assert np.all(np.abs(m[i] - mm) <= 4 * U * (b1 * np.abs(a[2]) + (1 - b1) * np.abs(a[1])))
            assert np.all(np.abs(v[i] - vv) <= 5 * U * vv + 1e-44)
            # the quotient of m and the root, whose own errors are those above: a handful of half steps each
            move = np.abs(lr / (1 - b1 ** t)) * (b1 * np.abs(a[2]) + (1 - b1) * np.abs(a[1])) / (np.sqrt(vv / (1 - b2 ** t)) + eps)
            assert np.all(np.abs(w[i] - ww) <= 3 * U * np.abs(old) + 20 * U * move + 1e-44)


def test_many_tensors(gt):
    """More than a launch takes, of all lengths, none among them; gradients that several tensors share; every tensor as by itself."""
    r = np.random.RandomState(0)
    sizes = [int(n) for n in np.exp(r.uniform(0, 8, 1100))]
    for n in (24, 25, 512, 513, 1100):
        w = [normal(i, s) for i, s in enumerate(sizes[:n])]
        g = normal(5, max(sizes))
        W, flat = views(gt, w), gt.gpu(g)
        G = [flat.narrow(1, 1, s) for s in sizes[:n]]
        opt = gt.optim.AdamW(W, G, weightDecay=0.3)
        for _ in range(2):
            opt.update()
        assert opt.step.float().tolist() == [2, 0]
        for i in list(range(0, n, 97)) + [n - 1]:
            alone, grad = gt.gpu(w[i]), gt.gpu(g[:sizes[i]])
            o = gt.optim.AdamW(alone, grad, weightDecay=0.3)
            o.update(); o.update()
            assert np.array_equal(alone.float(), W[i].float()) and np.array_equal(o.square[0].float(), opt.square[i].float())


def test_no_values(gt):
    for bits in (32, 8):
        opt = gt.optim.AdamW([], [], bits=bits)
        opt.update()
        assert opt.step.float().tolist() == [1, 0]
        w, g, empty = gt.gpu(normal(1, 300)), gt.gpu(normal(2, 300)), gt.GPUTensor()
        opt = gt.optim.AdamW([empty, w, empty], [gt.GPUTensor(), g, gt.GPUTensor()], bits=bits)
        opt.update()
        alone = gt.gpu(normal(1, 300))
        one = gt.optim.AdamW([gt.gpu(normal(1, 5)), alone], [gt.gpu(normal(2, 5)), g], bits=bits)
        one.update()
        assert np.array_equal(alone.float(), w.float())


def test_values_that_are_not_finite(gt):
    w, g = normal(1, 600), normal(2, 600)
    g[5], g[300], g[599] = np.nan, np.inf, 1e30
    W = gt.gpu(w)
    opt = gt.optim.AdamW(W, gt.gpu(g))
    opt.update()
    bad = ~np.isfinite(W.float())
    assert bad.nonzero()[0].tolist() == [5, 300]          # (1e30 squared is infinite: its step is none)
    W = gt.gpu(w)
    opt = gt.optim.AdamW(W, gt.gpu(g), bits=8)
    opt.update()
    m, v = (t[0].float() for t in opt.moments())
    # the blocks of the three values
    assert not np.isfinite(m[:256]).any() and not np.isfinite(v[:256]).any()
    assert not np.isfinite(m[256:512]).any() and not np.isfinite(v[256:512]).any() and not np.isfinite(v[512:]).any()
    assert np.isfinite(m[512:]).all() and (~np.isfinite(W.float())).nonzero()[0].tolist() == [5, 300]


# ------------------------------------------------------------------ 8 bits
B, TOP_M, TOP_S = F(2.0 ** -16), F(0.9375 - 2.0 ** -16), F(0.96875 - 2.0 ** -16)


def hashed(n, number, step, seed):
    mask = np.uint64(0xffffffff)
    key = ((seed & 0xffffffff) ^ (step * 0x9e3779b9 & 0xffffffff)) + number * 0x6a09e667
    h = (np.arange(n, dtype=np.uint64) * np.uint64(0x9e3779b9) + np.uint64(key & 0xffffffff)) & mask
    h = ((h ^ (h >> np.uint64(16))) * np.uint64(0xb7e15163)) & mask
    h = ((h ^ (h >> np.uint64(15))) * np.uint64(0xadf85459)) & mask
    return (h ^ (h >> np.uint64(16))).astype(np.int64)


def value(code, shift, scale):
    bits = (code.astype(np.int32) << shift) + np.int32(0x37800000)
    return (bits.view(F) - B) * scale


def coded(x, top, shift, noise, most):
    blocks = -(-x.size // 256)
    full = np.zeros(blocks * 256, F)
    full[:x.size] = x
    scale = full.reshape(blocks, 256).max(1) * (F(1) / top)
    scale = np.where(scale < F(2.0 ** -126), F(0), scale).astype(F)
    with np.errstate(divide="ignore"):
        inverse = np.where(scale == 0, F(0), F(1) / scale).astype(F)
    y = ((full.reshape(blocks, 256) * inverse[:, None]).reshape(-1) + B)[:x.size]
    bits = y.view(np.int32).astype(np.int64) - 0x37800000
    return np.minimum((bits + (noise << (shift - 16)) + (1 << (shift - 17))) >> shift, most), scale


class Eight:
    """The state of one tensor, stepped in FP32 operations one by one."""

    def __init__(self, n):
        self.n, blocks = n, -(-n // 256)
        self.m, self.r, self.scale_m, self.scale_r = np.zeros(n, np.int64), np.zeros(n, np.int64), np.zeros(blocks, F), np.zeros(blocks, F)

    def values(self):
        at = np.arange(self.n) // 256
        m = value(self.m & 127, 20, self.scale_m[at])
        return np.where(self.m & 128, -m, m), value(self.r, 19, self.scale_r[at])

    def step(self, g, b1, b2, number, step, seed):
        m, r = self.values()
        m = F(b1) * m + F(1 - b1) * g
        r = np.sqrt(F(b2) * (r * r) + F(1 - b2) * (g * g))
        h = hashed(self.n, number, step, seed)
        cm, self.scale_m = coded(np.abs(m), TOP_M, 20, h & 0xffff, 127)
        self.r, self.scale_r = coded(r, TOP_S, 19, h >> 16, 255)
        self.m = cm | (128 * (m < 0))
        return m, r


def state(opt, i, n):
    codes = [opt.meanCodes[i].float().view(np.uint8)[:n].astype(np.int64), opt.rootCodes[i].float().view(np.uint8)[:n].astype(np.int64)]
    return codes + list(opt.scales[i].float().reshape(-1, 2).T)


@pytest.mark.parametrize("b1,b2,seed,size", [(0.9, 0.999, 0, 1.0), (0.95, 0.9999, 12345678901, 1e-4), (0.0, 0.5, -3, 30.0), (0.9, 0.999, 7, 1e-25)])
@pytest.mark.parametrize("off", [0, 3])
def test_codes_are_those_of_the_definition(gt, b1, b2, seed, size, off):
    w = [normal(i, *s) for i, s in enumerate(SIZES)]
    W, G = views(gt, w, off), views(gt, w, off)
    opt = gt.optim.AdamW(W, G, learningRate=0.01, beta1=b1, beta2=b2, bits=8, seed=seed, weightDecay=0.1)
    like = [Eight(a.size) for a in w]
    r = np.random.RandomState(9)
    for t in range(1, 7):
        for i, s in enumerate(SIZES):
            g = (size * np.exp(2 * r.standard_normal(s)) * r.standard_normal(s) * (t != 4) * (r.random_sample(s) < 0.9)).astype(F)
            G[i].copy(g)
            like[i].g = g.reshape(-1)
        opt.update()
        means, squares = opt.moments()
        for i, s in enumerate(SIZES):
            n = like[i].n
            m, root = like[i].step(like[i].g, b1, b2, i, t, seed)
            for a, b, name in zip(state(opt, i, n), (like[i].m, like[i].r, like[i].scale_m, like[i].scale_r), ("mean codes", "root codes", "mean scales", "root scales")):
                assert np.array_equal(a, b), (t, i, name)
            kept, kept_root = like[i].values()
            assert means[i].size() == s and np.array_equal(means[i].float().reshape(-1), kept) and np.array_equal(squares[i].float().reshape(-1), kept_root * kept_root)
            # the weights' step is by the moments before they are rounded to codes
            old, new = w[i].reshape(-1).astype(np.float64), W[i].float().reshape(-1)
            move = 0.01 / (1 - b1 ** t) * m.astype(np.float64) / (root.astype(np.float64) / np.sqrt(1 - b2 ** t) + 1e-8)
            assert np.all(np.abs(new - (old * (1 - 0.01 * 0.1) - move)) <= 3 * U * np.abs(old) + 12 * U * np.abs(move) + 1e-44)
            w[i] = W[i].float()
    assert opt.step.float().tolist() == [6, 0]


def test_codes_of_many_values(gt):
    """So many that a block takes several turns at one tensor: the definition's codes all the same, in tensors whose ends lie anywhere in a turn."""
    sizes = [16 << 20, 2999999, 300, 2048 * 5, 8192 * 3 + 256]
    g = [normal(60 + i, n) * F(0.01) for i, n in enumerate(sizes)]
    W = [gt.GPUTensor(n).fill(0.0) for n in sizes]
    G = [gt.gpu(x) for x in g]
    opt = gt.optim.AdamW(W, G, bits=8, seed=5)
    like, w = [Eight(n) for n in sizes], [np.zeros(n) for n in sizes]
    for t in (1, 2):
        opt.update()
        for i, n in enumerate(sizes):
            m, root = like[i].step(g[i], 0.9, 0.999, i, t, 5)
            for a, b in zip(state(opt, i, n), (like[i].m, like[i].r, like[i].scale_m, like[i].scale_r)):
                assert np.array_equal(a, b)
            # as in test_codes_are_those_of_the_definition
            move = 1e-3 / (1 - 0.9 ** t) * m.astype(np.float64) / (root.astype(np.float64) / np.sqrt(1 - 0.999 ** t) + 1e-8)
            new = W[i].float().astype(np.float64)
            assert np.all(np.abs(new - (w[i] * (1 - 1e-5) - move)) <= 3 * U * np.abs(w[i]) + 12 * U * np.abs(move) + 1e-44)
            w[i] = new


def test_padding_codes_are_zero(gt):
    opt = gt.optim.AdamW(gt.gpu(normal(1, 300)), gt.gpu(normal(2, 300)), bits=8)
    opt.update()
    for t in (opt.meanCodes[0], opt.rootCodes[0]):
        assert not t.float().view(np.uint8)[300:].any()


def test_roots_follow_small_changes(gt):
    """Gradients stop: v falls by a thousandth of itself a step, less than its codes' distance.  Rounded at random its mean follows; a value's own error grows to some
    12 % (root of steps times their chance times the squared distance: 700 steps of 2^-7 times 2^-8, times 1/4 for the root's half), so the mean of 2^16 lies within
    5 of its errors, and 2 % for what the rounding adds to a square."""
    n = 1 << 16
    g = np.abs(normal(3, n)) + F(0.5)
    G = gt.gpu(g)
    opt = gt.optim.AdamW(gt.gpu(normal(1, n)), G, bits=8, beta2=0.999)
    opt.update()
    first = opt.moments()[1][0].float().astype(np.float64)
    G.zero()
    for _ in range(700):
        opt.update()
    v = opt.moments()[1][0].float().astype(np.float64)
    ratio = (v / first).mean() / 0.999 ** 700
    assert abs(ratio - 1) < 0.03


@pytest.mark.parametrize("bits", [32, 8])
def test_recorded_and_replayed(gt, bits):
    """A recorded update counts its steps, and keeps to the tensors' memory."""
    n = 5000
    w, g = normal(1, n), [normal(10 + i, n) for i in range(6)]
    alone, G = gt.gpu(w), gt.GPUTensor(n)
    opt = gt.optim.AdamW(alone, G, bits=bits)
    for t in g:
        G.copy(t)
        opt.update()
    want, moments = alone.float(), [t[0].float() for t in opt.moments()]
    stream = torch.cuda.Stream()
    gt.synchronize()
    gt.lib().THGPUSetStream(ctypes.c_void_p(stream.cuda_stream))
    try:
        W, G = gt.gpu(w), gt.gpu(g[0])
        opt = gt.optim.AdamW(W, G, bits=bits)
        opt.update()
        gt.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            opt.update()
        assert opt.step.float().tolist() == [1, 0]
        for t in g[1:]:
            G.copy(t)
            gt.synchronize()
            with torch.cuda.stream(stream):
                graph.replay()
            gt.synchronize()
        assert opt.step.float().tolist() == [6, 0]
        assert np.array_equal(W.float(), want)
        for a, b in zip(opt.moments(), moments):
            assert np.array_equal(a[0].float(), b)
        del graph
    finally:
        gt.synchronize()
        gt.lib().THGPUSetStream(None)


@pytest.mark.parametrize("bits", [32, 8])
def test_saved_and_continued(gt, bits):
    net = gt.nn.Linear(33, 20).gpu()
    W, G = net.getParameters()
    G.copy(normal(1, G.nElement()))
    opt = gt.optim.AdamW(W, G, bits=bits, seed=3)
    opt.update()
    twin = pickle.load(io.BytesIO(pickle.dumps(opt)))
    opt.update()
    twin.update()
    assert np.array_equal(opt.weights[0].float(), twin.weights[0].float())
    assert np.array_equal(opt.moments()[1][0].float(), twin.moments()[1][0].float()) and twin.step.float().tolist() == [2, 0]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("flat", [False, True])
def test_saved_with_its_module(gt, tmp_path, bits, flat):
    """After loading, and after the parameters have been brought into one storage, a step is one of the module's own tensors."""
    net = gt.nn.Sequential().add(gt.nn.Linear(33, 20)).add(gt.nn.LayerNorm(20)).gpu()
    params = gt.optim.parameters
    opt = gt.optim.AdamW(*params(net), bits=bits, seed=3)
    if flat:
        net.getParameters()
    for i, g in enumerate(params(net)[1]):
        g.copy(normal(i, *g.size()))
    opt.update()
    gt.save([net, opt], str(tmp_path / "both"))
    other, twin = gt.load(str(tmp_path / "both"))
    before = [t.float() for t in params(net)[0]]
    opt.update()
    twin.update()
    for a, b, c in zip(params(net)[0], params(other)[0], before):
        assert np.array_equal(a.float(), b.float()) and not np.array_equal(a.float(), c)


@pytest.mark.parametrize("bits", [32, 8])
def test_more_values_than_32_bits_count(gt, bits):
    """Both ends and the middle of one tensor of more than 2^31 values, as by themselves; the noise of a place counts on over 2^31."""
    n = 2 ** 31 + 2049 + 7
    W, G = gt.GPUTensor(n).fill(0.0), gt.GPUTensor(n).fill(0.0)
    for first, k in ((1, 300), (2 ** 31 - 100, 200), (n - 99, 100)):
        W.narrow(1, first, k).copy(normal(first % 1000, k)); G.narrow(1, first, k).copy(normal(first % 999, k))
    opt = gt.optim.AdamW(W, G, bits=bits)
    opt.update()
    for first, k in ((1, 300), (2 ** 31 - 100, 200), (n - 99, 100)):
        w, g = normal(first % 1000, k).astype(np.float64), normal(first % 999, k).astype(np.float64)
        want = w * (1 - 1e-5) - 1e-3 * g / (np.abs(g) + 1e-8)
        assert np.all(np.abs(W.narrow(1, first, k).float() - want) <= 3 * U * np.abs(w) + 20e-3 * U)
    assert opt.step.float().tolist() == [1, 0]
    if bits == 32:
        last = opt.mean[0].narrow(1, n - 99, 100).float()
        assert np.all(np.abs(last - 0.1 * normal((n - 99) % 999, 100).astype(np.float64)) <= 4 * U)
