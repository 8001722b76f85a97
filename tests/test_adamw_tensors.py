"""Which tensors optim.AdamW updates: each once, also where a module occurs twice; the fields of the other width's moments; the default seed."""
import inspect

import numpy as np
import pytest

import mcw_cppamp_torch_b200 as gt
from mcw_cppamp_torch_b200 import nn, optim
from test_feedforward_refusals import fake  # noqa: F401
from test_gpu_adamw import hashed
from test_routing_refusals import adamw


def test_weights_listed_again(fake):  # noqa: F811
    a, b, c, ga, gb = fake(7, 3), fake(256), fake(5), fake(7, 3), fake(256)
    empty = gt.GPUTensor()
    again = a.narrow(1, 1, 7)                            # another tensor over the same memory
    weights, gradients = optim._once((a, b, empty, again, c, empty, b), (ga, gb, empty, ga, gb.narrow(1, 1, 5), empty, gb))
    assert [id(t) for t in weights] == [id(t) for t in (a, b, empty, c, empty)]
    assert [t.data_ptr() for t in gradients] == [t.data_ptr() for t in (ga, gb, empty, gb, empty)]
    with pytest.raises(ValueError, match="tensors 2 and 3 are the same weights"):
        optim.AdamW([b, a, again], [gb, ga, fake(7, 3)])
    # the start of a tensor is another one; whether they share memory the call says
    assert len(optim._once((b, b.narrow(1, 1, 9)), (gb, gb.narrow(1, 1, 9)))[0]) == 2


def test_moments_of_the_other_width(fake):  # noqa: F811
    m = adamw(fake, 32)
    del m._lists["scales"], m._lists["meanCodes"]
    assert not hasattr(m, "scales") and getattr(m, "meanCodes", None) is None and hasattr(m, "mean")
    with pytest.raises(AttributeError, match="no scales"):
        m.scales


def test_noise_of_the_default_seed():
    """No place has the noise that a place near it had some steps before.  (Two times 2^12 hashes of 32 bits have 2^24 / 2^32 equal pairs by chance.)"""
    seed = inspect.signature(optim.AdamW).parameters["seed"].default
    noise = [hashed(4096, 0, step, seed) for step in range(1, 40)]
    for i, a in enumerate(noise):
        for b in noise[i + 1:i + 9]:
            assert len(np.intersect1d(a, b)) <= 2
    # a hash that does repeat is seen
    assert len(np.intersect1d(hashed(4096, 0, 1, 0), hashed(4096, 0, 2, 0))) == 4095


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_module_that_occurs_twice(bits):
    """Its tensors take one step, by the gradient that both occurrences have added to."""
    shared = nn.Linear(12, 12)
    net = nn.Sequential().add(shared).add(nn.ReLU()).add(shared).add(nn.Linear(12, 3)).gpu()
    weights, gradients = optim.parameters(net)
    assert len(weights) == 6
    opt = optim.AdamW(weights, gradients, bits=bits, seed=1)
    assert len(opt.weights) == len(opt.gradWeights) == 4
    r = np.random.RandomState(0)
    before = [w.float().astype(np.float64) for w in opt.weights]
    for g in opt.gradWeights:
        g.copy(r.standard_normal(g.size()).astype(np.float32))
    opt.update()
    for w, g, b in zip(opt.weights, opt.gradWeights, before):
        d = g.float().astype(np.float64)
        want = b * (1 - 1e-5) - 1e-3 * d / (np.abs(d) + 1e-8)
        assert np.all(np.abs(w.float() - want) <= 2.0 ** -24 * (3 * np.abs(b) + 0.02))
