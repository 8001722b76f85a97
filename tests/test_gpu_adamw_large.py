"""optim.AdamW with moments in 8 bits over more values than 32 bits count: codes, scales, what they stand for and the noise of each place, at both ends and in the middle."""
import numpy as np
import pytest

import test_gpu_adamw as small
from test_gpu_adamw import F, U, Eight, normal

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gt():
    import mcw_cppamp_torch_b200 as gt
    return gt


class Stretch(Eight):
    """Blocks that start at place `first` of a tensor."""

    def __init__(self, first, n):
        super().__init__(n)
        self.first = first

    def step(self, *args):
        whole, small.hashed = small.hashed, self.hashed
        try:
            return super().step(*args)
        finally:
            small.hashed = whole

    def hashed(self, n, number, step, seed):
        mask = 0xffffffff
        key = ((seed & mask) ^ (step * 0x9e3779b9 & mask)) + number * 0x6a09e667
        out = []
        for place in range(self.first, self.first + n):
            h = (place * 0x9e3779b9 + key) & mask
            h = ((h ^ h >> 16) * 0xb7e15163) & mask
            h = ((h ^ h >> 15) * 0xadf85459) & mask
            out.append(h ^ h >> 16)
        return np.array(out, np.int64)


def test_codes_of_places_beyond_32_bits(gt):
    n = 2 ** 31 + 2056                                    # the last block has eight values
    stretches = [Stretch(0, 512), Stretch(2 ** 31 - 512, 1024), Stretch(n - 8 - 256, 264)]
    # places that differ by 2^31 differ in their noise, and a stretch that starts at none is the plain definition's
    assert np.array_equal(Stretch(0, 40).hashed(40, 3, 7, 11), small.hashed(40, 3, 7, 11))
    assert not np.array_equal(Stretch(2 ** 31, 40).hashed(40, 0, 1, 5), small.hashed(40, 0, 1, 5))
    W, G = gt.GPUTensor(n).fill(0.0), gt.GPUTensor(n).fill(0.0)
    opt = gt.optim.AdamW(W, G, bits=8, seed=5, weightDecay=0.0)
    old = [np.zeros(s.n) for s in stretches]
    for t in (1, 2, 3):
        g = [normal(10 * t + i, s.n) for i, s in enumerate(stretches)]
        for s, x in zip(stretches, g):
            G.narrow(1, s.first + 1, s.n).copy(x)
        opt.update()
        for i, (s, x) in enumerate(zip(stretches, g)):
            m, root = s.step(x, 0.9, 0.999, 0, t, 5)
            block, blocks = s.first // 256, -(-s.n // 256)
            for codes, want in ((opt.meanCodes, s.m), (opt.rootCodes, s.r)):
                assert np.array_equal(codes[0].narrow(1, 64 * block + 1, 64 * blocks).float().view(np.uint8)[:s.n], want), (t, i)
            assert np.array_equal(opt.scales[0].narrow(1, 2 * block + 1, 2 * blocks).float().reshape(-1, 2), np.stack([s.scale_m, s.scale_r], 1)), (t, i)
            # as in the tests of smaller tensors; the first three steps have no floor, and these gradients no bound
            move = 1e-3 / (1 - 0.9 ** t) * m.astype(np.float64) / (root.astype(np.float64) / np.sqrt(1 - 0.999 ** t) + 1e-8)
            now = W.narrow(1, s.first + 1, s.n).float().astype(np.float64)
            assert np.all(np.abs(now - (old[i] - move)) <= 3 * U * np.abs(old[i]) + 16 * U * np.abs(move) + 1e-44), (t, i)
            old[i] = now
    # nothing has moved where the gradients are zero
    for first, k in ((512, 2048), (2 ** 31 + 512, 1000)):
        assert not W.narrow(1, first + 1, k).float().any()
    del W, G
    mean, square = (t[0] for t in opt.moments())
    for s in stretches:
        m, root = s.values()
        assert np.array_equal(mean.narrow(1, s.first + 1, s.n).float(), m) and np.array_equal(square.narrow(1, s.first + 1, s.n).float(), (root * root).astype(F))
    assert opt.step.float().tolist() == [3, 0]
