"""optim.AdamW with moments in 8 bits over many steps: how far values move whose gradients are far below the largest of their block."""
import numpy as np
import pytest

from test_gpu_adamw import F, U, Eight

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gt():
    import mcw_cppamp_torch_b200 as gt
    return gt


def most_of(b1, b2):
    """How many learning rates a step of Adam is at most, whatever the gradients: of m = (1 - b1) sum b1^i g_i and v = (1 - b2) sum b2^i g_i^2 Cauchy's inequality gives
    |m| <= (1 - b1) / sqrt((1 - b2) (1 - b1^2 / b2)) sqrt(v), and the bias corrections make it less; room for steady gradients, whose 1 the codes' noise may pass."""
    return max(2.0, (1 - b1) / np.sqrt((1 - b2) * (1 - b1 * b1 / b2))) if b1 * b1 < b2 else np.inf


def gradients(kind, rel, n, steps):
    """One value of each block with gradients of size 1, the others `rel` of that."""
    r = np.random.RandomState(1)
    size = np.full(n, rel)
    size[::256] = 1
    for t in range(steps):
        g = size * r.standard_normal(n)
        if kind == "seldom":
            g = np.where(r.random_sample(n) < 0.7, 0, g)
        g[::256] = np.where(g[::256] == 0, 1, g[::256])
        yield g.astype(F)


@pytest.mark.parametrize("kind", ["noise", "seldom"])
@pytest.mark.parametrize("rel", [1e-4, 1e-5, 1e-6, 1e-7])
def test_small_values_move_as_far_as_adam_moves_them(gt, rel, kind):
    """No step is longer than any gradients could make one of Adam's.  Once the first steps are past, steps are as long in the mean as exact ones, some 0.23 learning rates, with what the codes add:
    the mean's codes lie 2^-19 of the block's largest apart, or an eighth of the value; rounding up or down has half of that as its spread, and sum 0.9^2i = 5.3 of
    those, 1.15 codes in all, are over 2^-19 of the largest root at least: 1.15 times the 0.23 of the block's largest, or 0.15 of the value's own."""
    n, steps, lr = 4096, 300, 1e-3
    small = np.arange(n) % 256 != 0
    W, G = gt.GPUTensor(n).fill(0.0), gt.GPUTensor(n)
    opt = gt.optim.AdamW(W, G, learningRate=lr, weightDecay=0.0, bits=8, seed=5)
    was, late = np.zeros(n), []
    for t, g in enumerate(gradients(kind, rel, n, steps), 1):
        G.copy(g)
        opt.update()
        now = W.float().astype(np.float64)
        step = (now - was)[small] / lr
        # (the weight's own half step, of at most 1, in learning rates)
        assert np.abs(step).max() <= most_of(0.9, 0.999) * (1 + 16 * U) + 2 * U * np.abs(now).max() / lr, t
        if t > 16:
            late.append((step ** 2).mean())
        was = now
    # 0.23 and 0.27 of noise are 0.35; "seldom": the block's largest is steadier, with means of up to some 0.6 of its root
    assert np.sqrt(np.mean(late)) <= (0.5 if kind == "noise" else 0.75)


@pytest.mark.parametrize("b1,b2,seed", [(0.9, 0.999, 1), (0.95, 0.9999, 2), (0.9, 0.95, 3), (0.95, 0.9, 4), (0.0, 0.999, 5)])
@pytest.mark.parametrize("off", [0, 3])
def test_steps_are_those_of_the_definition(gt, b1, b2, seed, off):
    """Gradients over nine powers of ten, many of them zero: the codes' definition, and steps by roots of at least 2^-19 of the scale before, from where one gradient's share of v is a
    sixteenth at most, and at least as large as makes a step Adam's longest."""
    n, lr, eps = 3001, 0.01, 1e-12
    r = np.random.RandomState(seed)
    size = 10 ** r.uniform(-9, 0, n)
    room, G = gt.GPUTensor(n + off).fill(0.0), gt.GPUTensor(n)
    W = room.narrow(1, 1 + off, n)
    opt = gt.optim.AdamW(W, G, learningRate=lr, beta1=b1, beta2=b2, epsilon=eps, weightDecay=0.1, bits=8, seed=seed)
    like, old = Eight(n), np.zeros(n)
    bound = floored = 0
    for t in range(1, 41):
        g = (size * r.standard_normal(n) * (r.random_sample(n) < 0.5)).astype(F)
        G.copy(g)
        opt.update()
        scale = like.scale_r[np.arange(n) // 256].astype(np.float64)
        m, root = (x.astype(np.float64) for x in like.step(g, b1, b2, 0, t, seed))
        assert np.array_equal(opt.scales[0].float().reshape(-1, 2)[:, 1], like.scale_r)
        c1, c2 = 1 - b1 ** t, 1 - b2 ** t
        least = 2.0 ** -19 * scale if c2 >= 16 * (1 - b2) else 0 * scale
        share = np.abs(m) / c1 / most_of(b1, b2) * np.sqrt(c2)
        move = lr * m / c1 / (np.maximum(np.maximum(root, least), share) / np.sqrt(c2) + eps)
        bound += int((share > np.maximum(root, least)).sum())
        floored += int((least > np.maximum(root, share)).sum())
        new = W.float().astype(np.float64)
        # the weight's three roundings; those of the factors, the root, the quotient and its product: a handful each of half steps
        assert np.all(np.abs(new - (old * (1 - lr * 0.1) - move)) <= 3 * U * np.abs(old) + 16 * U * np.abs(move) + 1e-44), t
        old = new
    assert bound or b1 in (0.0, 0.95)
    assert floored or b2 in (0.95, 0.9)
