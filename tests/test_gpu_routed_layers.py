"""Router, Dispatch, GroupedLinear, Combine and AdamW together, as a routed feed-forward block that is trained: gradients against 64 bits and against differences,
recorded and replayed, from two threads, on another stream."""
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
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randn(shape, generator=g)


def up(gt, t):
    return gt.gpu(t.numpy())


def down(t):
    return torch.from_numpy(t.float())


class Routed:
    """x + sum_i p_i W2[e_i] silu(W1[e_i] norm(x) + b1[e_i]) + b2[e_i] over the k experts e_i that a product with norm(x) chooses."""

    def __init__(self, gt, width, inner, experts, k, normalize, seed=0):
        self.gt = gt
        self.norm, self.scores, self.router = gt.nn.LayerNorm(width), gt.nn.FusedLinear(width, experts), gt.nn.Router(k, normalize)
        self.out, self.first, self.second = gt.nn.Dispatch(experts), gt.nn.GroupedLinear(experts, width, inner, "silu"), gt.nn.GroupedLinear(experts, inner, width)
        self.join = gt.nn.Combine(width)
        self.layers = (self.norm, self.scores, self.first, self.second)
        for i, m in enumerate(self.layers):
            w, b = randn(seed + 2 * i, *m.weight.shape), 0.1 * randn(seed + 2 * i + 1, *m.bias.shape)
            m.weight, m.bias = (1 + 0.1 * w if i == 0 else w / m.weight.shape[-1] ** 0.5).numpy(), b.numpy()
            m.gpu()

    def zero(self):
        for m in self.layers:
            m.zeroGradParameters()

    def tensors(self):
        return [t for m in self.layers for t in (m.weight, m.bias)], [t for m in self.layers for t in (m.gradWeight, m.gradBias)]

    def forward(self, x, closed=None):
        self.x, h = x, self.norm.forward(x)
        s = self.scores.forward(h)
        if closed is not None:
            s.add(closed)
        self.s = s
        w, e = self.router.forward(s)
        rows, self.counts = self.out.forward([h, e])
        z = self.second.forward([self.first.forward([rows, self.counts]), self.counts])
        self.input = [z, w, self.out.positions, x]
        return self.join.forward(self.input)

    def backward(self, g):
        gz, gw, _, skip = self.join.backward(self.input, g)
        gi = self.first.backward([self.out.rows, self.counts], self.second.backward([self.first.output, self.counts], gz)[0])
        gh = self.out.backward([self.norm.output, self.router.output[1]], gi)[0]
        gh.add(self.scores.backward(self.norm.output, self.router.backward(self.s, gw)))
        return self.norm.backward(self.x, gh).add(skip)

    def exact(self, x, g, e, closed):
        """Output and gradients in 64 bits for the experts `e` that were chosen."""
        leaves = [t.requires_grad_() for t in [x.double()] + [down(t).double() for t in self.tensors()[0]]]
        X, nw, nb, rw, rb, w1, b1, w2, b2 = leaves
        h = torch.nn.functional.layer_norm(X, X.shape[-1:], nw, nb, self.norm.eps)
        s = h @ rw.t() + rb + (closed.double() if closed is not None else 0.0)
        on, at = e > 0, (e - 1).clamp(min=0)
        if self.router.normalize:
            p = torch.softmax(s.gather(1, at).masked_fill(~on, -torch.inf).masked_fill(~on.any(1, keepdim=True), 0.0), 1)
        else:
            p = torch.softmax(s.masked_fill(~on.any(1, keepdim=True), 0.0), 1).gather(1, at)
        p = p * on
        y = X
        for i in range(e.shape[1]):
            a = torch.nn.functional.silu(torch.einsum("ti,toi->to", h, w1[at[:, i]]) + b1[at[:, i]])
            y = y + (p[:, i, None] * (torch.einsum("ti,toi->to", a, w2[at[:, i]]) + b2[at[:, i]]))
        grads = torch.autograd.grad(y, leaves, g.double())
        return y.detach(), grads


def close(got, want, what, rel=4e-5):
    """Six chained FP32-accurate products: 2^-19 of their |products| each, which for sums of random signs is some 2^-19 root(terms) of the result's own size at
    most; against the result's norm, with the softmax's slope between them."""
    d, n = float((got.double() - want).norm()), float(want.norm())
    assert d <= rel * n, (what, d / n)


NAMES = ("input", "norm weight", "norm bias", "router weight", "router bias", "first weight", "first bias", "second weight", "second bias")


@pytest.mark.parametrize("tokens,width,inner,experts,k,normalize,padded", [(1, 64, 96, 4, 2, True, 0), (40, 64, 96, 8, 2, False, 5), (700, 128, 160, 16, 4, True, 0),
                                                                          (33, 75, 50, 5, 3, True, 7), (600, 64, 32, 30, 6, False, 100)])
def test_against_64_bits(gt, tokens, width, inner, experts, k, normalize, padded):
    b = Routed(gt, width, inner, experts, k, normalize)
    x, g = randn(20, tokens, width), randn(21, tokens, width)
    closed = None
    if padded:
        closed = torch.zeros(tokens, experts)
        closed[tokens - padded:] = -torch.inf
        closed[0, 1:] = -torch.inf                        # one open expert, fewer than k
    b.zero()
    y = down(b.forward(up(gt, x), None if closed is None else up(gt, closed)))
    gi = down(b.backward(up(gt, g)))
    e = down(b.router.output[1]).long()
    if padded:
        assert not e[tokens - padded:].any() and int((e[0] > 0).sum()) == 1
    want, grads = b.exact(x, g, e, closed)
    close(y, want, "output")
    for a, w, name in zip([gi] + [down(t) for t in b.tensors()[1]], grads, NAMES):
        close(a, w, name)


def test_differences(gt):
    """Gradients of sum(g y) against differences in the block's own outputs.  The other experts are closed while a weight moves: a token that changed its experts would
    not move by its gradient."""
    b = Routed(gt, 24, 40, 6, 2, True)
    x, g = randn(20, 8, 24), randn(21, 8, 24)
    b.zero()
    b.forward(up(gt, x))
    e = down(b.router.output[1])
    gi = down(b.backward(up(gt, g)))
    grads = [down(t) for t in b.tensors()[1]]
    h = 2.0 ** -8
    closed = up(gt, torch.full((8, 6), -torch.inf).scatter(1, e.long() - 1, 0.0))

    def loss(xv):
        y = (down(b.forward(up(gt, xv), closed)).double() * g.double()).sum()
        assert torch.equal(down(b.router.output[1]).sort(1).values, e.sort(1).values)
        return float(y)
    # the outputs' roundings (a few 2^-21 each of 192 values of size 1 to 3) over 2 h; third derivatives below 1000
    tol = 192 ** 0.5 * 10 * 2.0 ** -21 / (2 * h) + 1000 * h * h / 6
    for i, j in ((0, 0), (3, 11), (7, 23)):
        d = torch.zeros_like(x)
        d[i, j] = h
        assert abs((loss(x + d) - loss(x - d)) / (2 * h) - float(gi[i, j])) <= tol
    for t, grad in zip(b.tensors()[0], grads):
        w = down(t)
        for at in (0, w.numel() // 2, w.numel() - 1):
            v = []
            for sign in (1, -1):
                c = w.clone()
                c.view(-1)[at] += sign * h
                t.copy(c.numpy())
                v.append(loss(x))
            t.copy(w.numpy())
            assert abs((v[0] - v[1]) / (2 * h) - float(grad.view(-1)[at])) <= tol


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_of_training(gt, bits):
    """The update of all of a block's tensors is that of their gradients."""
    b = Routed(gt, 64, 96, 8, 2, True)
    opt = gt.optim.AdamW(*b.tensors(), learningRate=0.01, weightDecay=0.1, bits=bits)
    b.zero()
    b.forward(up(gt, randn(20, 50, 64)))
    b.backward(up(gt, randn(21, 50, 64)))
    before, grads = [down(t).double() for t in b.tensors()[0]], [down(t).double() for t in b.tensors()[1]]
    opt.update()
    for w, g, t in zip(before, grads, b.tensors()[0]):
        want = w * (1 - 0.001) - 0.01 * g / (g.abs() + 1e-8)
        assert torch.all((down(t).double() - want).abs() <= 2.0 ** -24 * (3 * w.abs() + 0.2))


def test_recorded_and_replayed(gt):
    """What follows the dispatch, in two recordings replayed in turn over other inputs.  Dispatch itself says that it cannot be recorded, and spoils nothing."""
    tokens, width, experts, k = 60, 96, 6, 2
    stream = torch.cuda.Stream()
    gt.synchronize()
    gt.lib().THGPUSetStream(ctypes.c_void_p(stream.cuda_stream))
    try:
        b = Routed(gt, width, 64, experts, k, True)
        X, G = up(gt, randn(20, tokens, width)), up(gt, randn(21, tokens, width))
        b.forward(X)
        b.zero()
        b.backward(G)
        h, e, w = b.norm.output, b.router.output[1], b.router.output[0]

        def there():
            b.router.forward(b.s)
            b.join.forward(b.input)

        def back():
            b.zero()
            return b.backward(G)
        for _ in range(2):
            there(); back()
        gt.synchronize()
        graphs = []
        for f in (there, back):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                f()
                if f is there:
                    with pytest.raises(gt.THCError, match="cannot be recorded"):
                        b.out.forward([h, e])

        def results():
            return [down(t) for t in [b.join.output, b.norm.gradInput, w] + b.tensors()[1]]
        for seed in (1, 2, 3):
            b.second.output.copy(randn(seed, *b.second.output.size()).numpy())
            G.copy(randn(seed + 10, tokens, width).numpy())
            there(); back()
            want = results()
            for t in (b.join.output, b.norm.gradInput, b.first.gradWeight, w):
                t.fill(float("nan"))
            gt.synchronize()
            with torch.cuda.stream(stream):
                graphs[0].replay()
                graphs[1].replay()
            gt.synchronize()
            for a, c in zip(results(), want):
                assert torch.equal(a, c)
            up(gt, randn(30, 700, width))
            other = gt.nn.Dispatch(experts)            # a call between the replays
            other.forward([up(gt, randn(30, 700, width)), gt.gpu(np.ones((700, 4), np.float32))])
        del graphs
    finally:
        gt.synchronize()
        gt.lib().THGPUSetStream(None)


def test_two_threads(gt):
    """Two threads, each on its own stream of the device, at the same time: the results of each alone."""
    def work(out, seed):
        try:
            b = Routed(gt, 64, 96, 8, 2, True, seed)
            opt = gt.optim.AdamW(*b.tensors(), bits=8, seed=seed)
            for i in range(8):
                b.zero()
                y = down(b.forward(up(gt, randn(seed + i, 900 if i % 2 else 30, 64))))
                gi = down(b.backward(up(gt, randn(seed + i + 50, 900 if i % 2 else 30, 64))))
                opt.update()
                out.append([y, gi, torch.from_numpy(b.counts)] + [down(t) for t in b.tensors()[0]])
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
        assert len(a) == len(b) == 8, (a[-1], b[-1])
        for p, q in zip(a, b):
            assert all(torch.equal(u, v) for u, v in zip(p, q))


def test_modules_are_saved_and_cloned(gt):
    b = Routed(gt, 32, 16, 4, 2, True)
    x, g = up(gt, randn(1, 9, 32)), up(gt, randn(2, 9, 32))
    b.zero()
    y = down(b.forward(x))
    b.backward(g)
    router, out, join = b.router.clone(), b.out.clone(), b.join.clone()
    assert torch.equal(down(join.forward(b.input)), y) and len(join.gradInput) == 3
    w, e = router.forward(b.s)
    rows, counts = out.forward([b.norm.output, e])
    assert torch.equal(down(rows), down(b.out.rows)) and np.array_equal(counts, b.counts)
    again = b.join.clone()
    assert torch.equal(down(again.backward(b.input, g)[1]), down(b.join.gradWeights))
