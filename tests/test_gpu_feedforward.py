"""LayerNorm, FusedLinear and GroupedLinear together, as a feed-forward block and as a routed one: gradients against float64 and against
differences, recorded and replayed, from two threads, on another stream, over more values than 32 bits count."""
import ctypes
import threading

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


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


class Block:
    """x + W2 gelu(W1 norm(x) + b1) + b2, the skip connection in the second product's epilogue."""

    def __init__(self, gt, width, inner, seed=0):
        self.gt = gt
        self.norm, self.up, self.down = gt.nn.LayerNorm(width), gt.nn.FusedLinear(width, inner, "gelu"), gt.nn.FusedLinear(inner, width)
        for i, (m, fan) in enumerate(((self.norm, 0), (self.up, width), (self.down, inner))):
            w, b = randn(seed + 2 * i, *m.weight.shape), 0.1 * randn(seed + 2 * i + 1, *m.bias.shape)
            m.weight, m.bias = (1 + 0.1 * w if not fan else w / fan ** 0.5).cpu().numpy(), b.cpu().numpy()
            m.gpu()
        self.modules = (self.norm, self.up, self.down)

    def forward(self, x):
        self.x = x
        return self.down.forward([self.up.forward(self.norm.forward(x)), x])

    def backward(self, g):
        gi, skip = self.down.backward([self.up.output, self.x], g)
        gi = self.norm.backward(self.x, self.up.backward(self.norm.output, gi))
        return gi.add(skip)

    def zero(self):
        for m in self.modules:
            m.zeroGradParameters()

    def exact(self, x, g):
        leaves = [x.double()] + [down(t).double() for m in self.modules for t in (m.weight, m.bias)]
        leaves = [t.requires_grad_() for t in leaves]
        x, w, b, w1, b1, w2, b2 = leaves
        h = torch.nn.functional.layer_norm(x, x.shape[-1:], w, b, self.norm.eps)
        y = x + torch.nn.functional.gelu(h @ w1.t() + b1) @ w2.t() + b2
        return y.detach(), torch.autograd.grad(y, leaves, g.double())


def close(got, want, what, rel=2e-5):
    """A few chained FP32-accurate products: 2^-19 of their |products| each, which for sums of random signs is some 2^-19 root(terms) of the
    result's own size at most; against the result's norm."""
    d, n = float((got.double() - want).norm()), float(want.norm())
    assert d <= rel * n, (what, d / n)


@pytest.mark.parametrize("rows,width,inner", [(1, 64, 96), (5, 512, 1000), (300, 768, 2048), (2048, 1024, 4096), (33, 257, 131)])
def test_block(gt, rows, width, inner):
    block, x, g = Block(gt, width, inner), randn(10, rows, width), randn(11, rows, width)
    block.zero()
    y = down(block.forward(up(gt, x)))
    gi = down(block.backward(up(gt, g)))
    want, grads = block.exact(x, g)
    close(y, want, "output")
    got = [gi] + [down(t) for m in block.modules for t in (m.gradWeight, m.gradBias)]
    for a, b, name in zip(got, grads, ("input", "norm weight", "norm bias", "first weight", "first bias", "second weight", "second bias")):
        close(a, b, name)


def test_differences(gt):
    """The block's gradients against differences of sum(g * y) in its own outputs."""
    block, x, g = Block(gt, 48, 80), randn(10, 6, 48), randn(11, 6, 48)
    block.zero()
    block.forward(up(gt, x))
    gi = down(block.backward(up(gt, g)))
    gw = down(block.up.gradWeight)

    def loss(xv):
        return float((down(block.forward(up(gt, xv))).double() * g.double()).sum())
    h = 2.0 ** -6
    # the outputs' roundings (a few 2^-21 each of 288 values of size 1 to 3) over 2h; third derivatives below 100
    tol = 288 ** 0.5 * 10 * 2.0 ** -21 / (2 * h) + 100 * h * h / 6
    for i, j in ((0, 0), (2, 17), (5, 47)):
        d = torch.zeros_like(x)
        d[i, j] = h
        assert abs((loss(x + d) - loss(x - d)) / (2 * h) - float(gi[i, j])) <= tol
    w = down(block.up.weight)
    for i, j in ((0, 0), (40, 7), (79, 47)):
        d = torch.zeros_like(w)
        d[i, j] = h
        block.up.weight.copy((w + d).cpu().numpy())
        hi = loss(x)
        block.up.weight.copy((w - d).cpu().numpy())
        lo = loss(x)
        block.up.weight.copy(w.cpu().numpy())
        assert abs((hi - lo) / (2 * h) - float(gw[i, j])) <= tol


@pytest.mark.parametrize("tokens,groups,width,inner", [(40, 4, 64, 96), (1000, 8, 256, 320), (17, 30, 128, 100)])
def test_routed_block(gt, tokens, groups, width, inner):
    """Rows to their experts by index, through two grouped layers, and back by indexCopy."""
    rs = np.random.RandomState(tokens)
    expert = rs.randint(0, groups, tokens)
    order = np.argsort(expert, kind="stable")
    counts = np.bincount(expert, minlength=groups)
    first, second = gt.nn.GroupedLinear(groups, width, inner, "silu"), gt.nn.GroupedLinear(groups, inner, width)
    for i, m in enumerate((first, second)):
        m.weight, m.bias = (randn(2 * i, *m.weight.shape) / m.weight.shape[2] ** 0.5).cpu().numpy(), randn(2 * i + 1, *m.bias.shape).cpu().numpy()
        m.gpu().zeroGradParameters()
    x, g = randn(10, tokens, width), randn(11, tokens, width)
    xs = up(gt, x).index(1, order + 1)
    y = second.forward([first.forward([xs, counts]), counts])
    out = down(gt.GPUTensor(tokens, width).indexCopy(1, order + 1, y))
    gs = up(gt, g).index(1, order + 1)
    gi = first.backward([xs, counts], second.backward([first.output, counts], gs)[0])[0]
    gx = down(gt.GPUTensor(tokens, width).indexCopy(1, order + 1, gi))
    leaves = [t.double().requires_grad_() for t in (x, down(first.weight), down(first.bias), down(second.weight), down(second.bias))]
    X, w1, b1, w2, b2 = leaves
    e = torch.from_numpy(expert).cuda()
    h = torch.nn.functional.silu(torch.einsum("ti,toi->to", X, w1[e]) + b1[e])
    want = torch.einsum("ti,toi->to", h, w2[e]) + b2[e]
    close(out, want.detach(), "output")
    grads = torch.autograd.grad(want, leaves, g.double())
    for a, b, name in zip([gx] + [down(t) for m in (first, second) for t in (m.gradWeight, m.gradBias)], grads, ("input", "w1", "b1", "w2", "b2")):
        close(a, b, name)


def wrap(gt, t):
    L = gt.lib()
    s = L.THGPUStorage_newWithData(t.data_ptr(), t.numel())
    v = gt.GPUTensor(_ptr=L.THGPUTensor_newWithStorage1d(s, 0, t.numel(), 1)).view(*t.shape)
    L.THGPUStorage_free(s)
    return v


@pytest.mark.parametrize("rows,width,inner", [(3, 256, 512), (600, 1024, 2048), (40, 10000, 64)])
def test_recorded_and_replayed(gt, rows, width, inner):
    """A block and a grouped layer in two recordings, replayed in turn over other inputs, with other work between them."""
    block = Block(gt, width, inner)
    experts = gt.nn.GroupedLinear(5, width, inner, "silu").gpu()
    counts = [rows // 3, 0, rows - rows // 3 - 1, 1, 0]
    x, g, ge = torch.zeros(rows, width, device="cuda"), torch.zeros(rows, width, device="cuda"), torch.zeros(rows, inner, device="cuda")
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    gt.lib().THGPUSetStream(ctypes.c_void_p(stream.cuda_stream))
    try:
        X, G, GE = wrap(gt, x), wrap(gt, g), wrap(gt, ge)

        def one():
            block.zero()
            block.forward(X)
            block.result = block.backward(G)

        def two():
            experts.zeroGradParameters()
            experts.forward([X, counts])
            experts.backward([X, counts], GE)

        def results():
            return [down(t).clone() for t in (block.down.output, block.result, block.norm.gradWeight, block.up.gradWeight, block.down.gradBias, experts.output,
                                              experts.gradInput[0], experts.gradWeight, experts.gradBias)]
        for _ in range(2):
            one(); two()
        gt.synchronize()
        graphs = []
        for f in (one, two):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                f()
        for seed in (1, 2, 3):
            x.copy_(randn(seed, rows, width)); g.copy_(randn(seed + 10, rows, width)); ge.copy_(randn(seed + 20, rows, inner))
            torch.cuda.synchronize()
            one(); two()
            gt.synchronize()
            want = results()
            for t in (block.down.output, experts.output, block.up.gradWeight, experts.gradWeight):
                t.fill(float("nan"))
            gt.synchronize()
            with torch.cuda.stream(stream):
                graphs[seed % 2].replay()
                graphs[1 - seed % 2].replay()
            gt.synchronize()
            for a, b in zip(results(), want):
                assert torch.equal(a, b)
        del graphs
    finally:
        gt.synchronize()
        gt.lib().THGPUSetStream(None)


@pytest.mark.parametrize("groups,most", [(12, 3), (12, 9), (500, 3), (500, 9), (500, 40)])
def test_routed_layers_recorded_and_replayed(gt, groups, most):
    """Lists of groups that travel with a launch and that lie in memory, rows of a group few and not; other counts between the replays."""
    m = gt.nn.GroupedLinear(groups, 72, 600, "gelu").gpu()
    counts, others = np.arange(groups) % most, (np.arange(groups) * 5 + 1) % (most + 3)
    rows, more = int(counts.sum()), int(others.sum())
    x, g = torch.zeros(rows, 72, device="cuda"), torch.zeros(rows, 600, device="cuda")
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    gt.lib().THGPUSetStream(ctypes.c_void_p(stream.cuda_stream))
    try:
        X, G, X2, G2 = wrap(gt, x), wrap(gt, g), up(gt, randn(5, more, 72)), up(gt, randn(6, more, 600))

        def step():
            m.zeroGradParameters()
            m.forward([X, counts])
            m.backward([X, counts], G)

        def results():
            return [down(t).clone() for t in (m.output, m.gradInput[0], m.gradWeight, m.gradBias)]
        for _ in range(2):
            step()
        gt.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        kept = (m.output, m.gradInput, m.preactivation, m.gradPreactivation)
        for seed in (1, 2):
            x.copy_(randn(seed, rows, 72)); g.copy_(randn(seed + 10, rows, 600))
            torch.cuda.synchronize()
            step()
            gt.synchronize()
            want = results()
            m.output, m.gradInput, m.preactivation, m.gradPreactivation = (gt.GPUTensor() for _ in range(4))
            m.forward([X2, others])
            m.backward([X2, others], G2)
            m.output, m.gradInput, m.preactivation, m.gradPreactivation = kept
            m.gradWeight.fill(float("nan")); m.output.fill(float("nan"))
            gt.synchronize()
            with torch.cuda.stream(stream):
                graph.replay()
            gt.synchronize()
            for a, b in zip(results(), want):
                assert torch.equal(a, b)
        del graph
    finally:
        gt.synchronize()
        gt.lib().THGPUSetStream(None)


def test_two_threads(gt):
    """Two threads, each on its own stream of the device, at the same time: the results of each alone."""
    def work(out, seed):
        try:
            block = Block(gt, 512, 1024, seed)
            for k in range(6):
                x, g = randn(seed + k, 300, 512), randn(seed + k + 50, 300, 512)
                block.zero()
                y = down(block.forward(up(gt, x)))
                gi = down(block.backward(up(gt, g)))
                out.append((y, gi, down(block.up.gradWeight), down(block.norm.gradWeight)))
        except Exception as e:      # (a thread's exception would otherwise be lost)
            out.append(e)
    alone, both = ([], []), ([], [])
    for i in range(2):
        work(alone[i], 100 * i)
    threads = [threading.Thread(target=work, args=(both[i], 100 * i)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(alone, both):
        assert len(a) == len(b) == 6
        for p, q in zip(a, b):
            assert all(torch.equal(u, v) for u, v in zip(p, q))


def test_modules_are_saved_and_cloned(gt):
    net = gt.nn.Sequential().add(gt.nn.LayerNorm(32)).add(gt.nn.FusedLinear(32, 16, "silu")).gpu()
    x = up(gt, randn(1, 9, 32))
    y = down(net.forward(x))
    twin = net.clone()
    assert torch.equal(down(twin.forward(x)), y)
    w, g = net.getParameters()
    assert w.nElement() == 32 * 2 + 32 * 16 + 16
    assert torch.equal(down(net.forward(x)), y)
    experts = gt.nn.GroupedLinear(3, 32, 8, "gelu").gpu()
    a = down(experts.forward([x, [4, 0, 5]]))
    experts.getParameters()
    assert torch.equal(down(experts.clone().forward([x, [4, 0, 5]])), a)


# ------------------------------------------------------------------ more values than 32 bits count
@pytest.mark.parametrize("rows,size", [(262150, 8192), (70001, 32768), (2 ** 31 // 100 + 9, 100)])
def test_norm_over_large_tensors(gt, rows, size):
    m = gt.nn.LayerNorm(size).gpu()
    m.weight.copy((1 + 0.1 * randn(5, size)).cpu().numpy())
    x, g = gt.GPUTensor(rows, size).fill(1.0), gt.GPUTensor(rows, size).fill(0.0)
    xs, gs = randn(1, 4, size), randn(2, 4, size)
    for t, v in ((x, xs), (g, gs)):
        t.narrow(1, 1, 2).copy(v[:2].cpu().numpy())
        t.narrow(1, rows - 1, 2).copy(v[2:].cpu().numpy())
    small = gt.nn.LayerNorm(size).gpu()
    small.weight.copy(m.weight)
    want, wg = down(small.forward(up(gt, xs))), down(small.backward(up(gt, xs), up(gt, gs)))
    out = m.forward(x)
    assert torch.equal(torch.cat([down(out.narrow(1, 1, 2)), down(out.narrow(1, rows - 1, 2))]), want)
    assert float(out.narrow(1, 3, 1).sum()) == 0 and float(out.narrow(1, rows - 2, 1).sum()) == 0
    gi = m.backward(x, g)
    assert torch.equal(torch.cat([down(gi.narrow(1, 1, 2)), down(gi.narrow(1, rows - 1, 2))]), wg)
    want = down(small.gradWeight).double()
    assert torch.all((down(m.gradWeight).double() - want).abs() <= 2.0 ** -20 * 40)


@pytest.mark.parametrize("grouped", [False, True])
def test_linear_over_large_results(gt, grouped):
    """An output of more than 2^31 values, from rows that differ at both ends."""
    rows, inputs, outputs = 530000, 32, 4100
    m = (gt.nn.GroupedLinear(2, inputs, outputs, "gelu") if grouped else gt.nn.FusedLinear(inputs, outputs, "gelu")).gpu()
    few = (gt.nn.GroupedLinear(2, inputs, outputs, "gelu") if grouped else gt.nn.FusedLinear(inputs, outputs, "gelu")).gpu()
    few.weight.copy(m.weight); few.bias.copy(m.bias)
    x = gt.GPUTensor(rows, inputs).fill(0.5)
    xs = randn(1, 6, inputs)
    x.narrow(1, 1, 3).copy(xs[:3].cpu().numpy())
    x.narrow(1, rows - 2, 3).copy(xs[3:].cpu().numpy())
    out = m.forward([x, [100, rows - 100]] if grouped else x)
    want = down(few.forward([up(gt, xs), [3, 3]] if grouped else up(gt, xs))).double()
    got = torch.cat([down(out.narrow(1, 1, 3)), down(out.narrow(1, rows - 2, 3))]).double()
    assert torch.all((got - want).abs() <= 2.0 ** -17 * (1 + want.abs()))
    m.gradInput = gt.GPUTensor()
    g = gt.GPUTensor(rows, outputs).fill(0.0)
    gs = randn(2, 6, outputs)
    g.narrow(1, 1, 3).copy(gs[:3].cpu().numpy())
    g.narrow(1, rows - 2, 3).copy(gs[3:].cpu().numpy())
    m.zeroGradParameters(); few.zeroGradParameters()
    gi = m.backward([x, [100, rows - 100]] if grouped else x, g)
    wi = few.backward([up(gt, xs), [3, 3]] if grouped else up(gt, xs), up(gt, gs))
    if grouped:
        gi, wi = gi[0], wi[0]
    got = torch.cat([down(gi.narrow(1, 1, 3)), down(gi.narrow(1, rows - 2, 3))]).double()
    scale = 2.0 ** -17 * float(gs.abs().max()) * outputs ** 0.5
    assert torch.all((got - down(wi).double()).abs() <= scale)
    assert torch.all((down(m.gradWeight).double() - down(few.gradWeight).double()).abs() <= 2.0 ** -17 * 6 * 16)
