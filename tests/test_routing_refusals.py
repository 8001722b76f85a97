"""What Router, Dispatch, Combine and AdamW refuse, before any device is touched: tensors here are shapes over memory that nothing reads."""
import ctypes as C

import numpy as np
import pytest

import mcw_cppamp_torch_b200 as gt
from mcw_cppamp_torch_b200 import nn, optim
from mcw_cppamp_torch_b200._lib import TP
from test_feedforward_refusals import fake  # noqa: F401


def router(fake, k=2, normalize=True):  # noqa: F811
    m = nn.Router(k, normalize)
    m.output, m.gradInput = [fake(5, k), fake(5, k)], fake(5, 6)
    return m


def test_router(fake):  # noqa: F811
    x, w, e = fake(5, 6), fake(5, 2), fake(5, 2)
    for k in (0, -1):
        with pytest.raises(ValueError):
            nn.Router(k)
    with pytest.raises(TypeError):
        router(fake).forward(np.zeros((5, 6), np.float32))
    with pytest.raises(gt.THCError, match="Invalid argument 1: batch"):
        router(fake).forward(fake(5, 6, 2))
    with pytest.raises(gt.THCError, match="1024 scores"):
        router(fake).forward(fake(5, 1025))
    for k, size in ((7, 6), (33, 64)):
        with pytest.raises(gt.THCError, match="Invalid argument 4: between 1 and 32"):
            router(fake, k).forward(fake(5, size))
    with pytest.raises(gt.THCError, match="Invalid argument 4: between 1 and 32"):
        gt.lib().THGPUNN_Router_updateOutput(x._p, w._p, e._p, 0, 1)
    for i, bad, match in ((0, x, "shares memory"), (1, x, "shares memory"), (0, fake(5, 2, strides=(3, 1)), "contiguous result")):
        m = router(fake)
        m.output[i] = bad
        with pytest.raises(gt.THCError, match=match):
            m.forward(x)
    m = router(fake)
    m.output[1] = m.output[0]
    with pytest.raises(gt.THCError, match="shares memory"):
        m.forward(x)
    for bad in (fake(5, 3), fake(4, 2), fake(10)):
        with pytest.raises(gt.THCError, match="gradWeights has the wrong size"):
            router(fake).backward(x, bad)
    for i, bad in ((0, fake(4, 2)), (1, fake(5, 3)), (0, fake(5, 2, strides=(3, 1))), (1, fake(5, 2, strides=(1, 5)))):
        m = router(fake)
        m.output[i] = bad
        with pytest.raises(gt.THCError, match="as updateOutput left them"):
            m.backward(x, fake(5, 2))
    m = router(fake)
    m.gradInput = m.output[0]
    with pytest.raises(gt.THCError, match="shares memory"):
        m.backward(x, fake(5, 2))
    m = router(fake)
    m.gradInput = None
    assert m.backward(x, fake(5, 2)) is None


def dispatch(fake):  # noqa: F811
    m = nn.Dispatch(4)
    m.rows, m.positions, m.gradRows = fake(10, 6), fake(5, 2), fake(5, 6)
    return m


def test_dispatch(fake):  # noqa: F811
    with pytest.raises(ValueError):
        nn.Dispatch(0)
    x, e = fake(5, 6), fake(5, 2)
    with pytest.raises(TypeError):
        dispatch(fake).forward([x, np.ones((5, 2), np.float32)])
    with pytest.raises(gt.THCError, match="Invalid argument 1: matrix of rows"):
        dispatch(fake).forward([fake(5, 3, 2), e])
    with pytest.raises(gt.THCError, match="Invalid argument 2: matrix of a row of slots"):
        dispatch(fake).forward([x, fake(5)])
    for bad in (fake(4, 2), fake(6, 2)):
        with pytest.raises(gt.THCError, match="Invalid argument 2: a row of slots"):
            dispatch(fake).forward([x, bad])
    with pytest.raises(gt.THCError, match="2.24 slots"):
        dispatch(fake).forward([fake(2 ** 24 + 1, 1, strides=(0, 1)), fake(2 ** 24 + 1, 1, strides=(0, 1))])
    with pytest.raises(gt.THCError, match="2.23 values"):
        dispatch(fake).forward([fake(1, 2 ** 23 + 1, strides=(0, 0)), fake(1, 1)])
    m = nn.Dispatch(4097)
    with pytest.raises(gt.THCError, match="4096 groups"):
        m.forward([x, e])
    for name, bad in (("rows", x), ("rows", e), ("positions", x), ("positions", e)):
        m = dispatch(fake)
        setattr(m, name, bad)
        with pytest.raises(gt.THCError, match="shares memory"):
            m.forward([x, e])
    m = dispatch(fake)
    m.positions = m.rows.narrow(1, 1, 5).narrow(2, 1, 2)
    with pytest.raises(gt.THCError, match="shares memory"):
        m.forward([x, e])
    L = gt.lib()
    rows, positions = fake(10, 6), fake(5, 2)
    with pytest.raises(gt.THCError, match="room for a count"):
        L.cdll.THGPUNN_Dispatch_updateOutput.argtypes, kept = None, L.cdll.THGPUNN_Dispatch_updateOutput.argtypes
        try:
            L.cdll.THGPUNN_Dispatch_updateOutput(x._p, e._p, rows._p, positions._p, None, 4)
        finally:
            L.cdll.THGPUNN_Dispatch_updateOutput.argtypes = kept
        message = L.THGPUGetLastError().decode()
        L.THGPUClearError()
        raise gt.THCError(message)
    frozen = np.zeros(4, np.int64)
    frozen.flags.writeable = False
    for bad in (frozen, np.zeros(4, np.int32), [0, 0, 0, 0]):
        with pytest.raises((C.ArgumentError, TypeError)):
            L.THGPUNN_Dispatch_updateOutput(x._p, e._p, rows._p, positions._p, bad, 4)
    for bad in (fake(10, 5), fake(11, 6)):
        with pytest.raises(gt.THCError, match="gradOutput has the wrong size"):
            dispatch(fake).backward([x, e], [bad, None])
    m = dispatch(fake)
    m.positions = fake(4, 2)
    with pytest.raises(gt.THCError, match="as updateOutput left them"):
        m.backward([x, e], fake(8, 6))
    m = dispatch(fake)
    g = fake(8, 6)
    m.gradRows = g.narrow(1, 1, 5)
    with pytest.raises(gt.THCError, match="shares memory"):
        m.backward([x, e], g)


def combine(fake):  # noqa: F811
    m = nn.Combine()
    m.output, m.gradRows, m.gradWeights = fake(5, 6), fake(8, 6), fake(5, 2)
    return m


def test_combine(fake):  # noqa: F811
    z, w, p, r, g = fake(8, 6), fake(5, 2), fake(5, 2), fake(5, 6), fake(5, 6)
    with pytest.raises(ValueError, match="matrix of rows"):
        nn.Combine().forward([gt.GPUTensor(), w, p])
    with pytest.raises(ValueError, match="matrix of rows"):
        combine(fake).forward([fake(48), w, p])
    for bad in (fake(5, 3), fake(4, 2), fake(10)):
        with pytest.raises(gt.THCError, match="Invalid argument 2: a weight for each slot"):
            combine(fake).forward([z, bad, p])
        with pytest.raises(gt.THCError, match="Invalid argument 2: a weight for each slot"):
            combine(fake).backward([z, bad, p], g)
    with pytest.raises(gt.THCError, match="Invalid argument 3"):
        combine(fake).forward([z, None, fake(5)])
    for bad in (fake(5, 7), fake(4, 6)):
        with pytest.raises(gt.THCError, match="residual"):
            combine(fake).forward([z, w, p, bad])
    with pytest.raises(gt.THCError, match="rows of the given size"):
        m = combine(fake)
        m.size = 7
        m.forward([z, w, p])
    for size in (0, -1, 2 ** 23 + 1):
        with pytest.raises(gt.THCError, match="size must be"):
            gt.lib().THGPUNN_Combine_updateOutput(z._p, w._p, p._p, None, r._p, size)
    for bad in (z, w, p, r):
        m = combine(fake)
        m.output = bad
        with pytest.raises(gt.THCError, match="shares memory"):
            m.forward([z, w, p, r])
    for name, bad in (("gradRows", z), ("gradRows", g), ("gradWeights", w), ("gradWeights", p)):
        m = combine(fake)
        setattr(m, name, bad)
        with pytest.raises(gt.THCError, match="shares memory"):
            m.backward([z, w, p], g)
    m = combine(fake)
    m.gradRows = fake(8, 6, strides=(7, 1))
    with pytest.raises(gt.THCError, match="contiguous result"):
        m.backward([z, w, p], g)
    for bad in (fake(4, 6), fake(30)):
        with pytest.raises(gt.THCError, match="Invalid argument 4"):
            combine(fake).backward([z, w, p], bad)
    with pytest.raises(gt.THCError, match="rows of gradOutput's size"):
        combine(fake).backward([z, w, p], fake(5, 7))
    with pytest.raises(gt.THCError, match="Invalid argument 6: weights have a gradient"):
        m = combine(fake)
        gt.lib().THGPUNN_Combine_backward(z._p, None, p._p, g._p, m.gradRows._p, m.gradWeights._p)


def test_combine_saves_no_caller_tensor(fake):  # noqa: F811
    m = combine(fake)
    m.gradInput = [m.gradRows, m.gradWeights, None, fake(5, 6)]
    assert m.__getstate__()["gradInput"] == [m.gradRows, m.gradWeights, None]


def adamw(fake, bits=32, sizes=((7, 3), (256,), (300,))):  # noqa: F811
    m = object.__new__(optim.AdamW)
    m.__dict__.update(learningRate=1e-3, beta1=0.9, beta2=0.999, epsilon=1e-8, weightDecay=0.01, bits=bits, seed=0, step=fake(2), _lists={})
    m.weights, m.gradWeights = ([fake(*s) for s in sizes] for _ in range(2))
    n = [int(np.prod(s)) for s in sizes]
    blocks = [-(-k // 256) for k in n]
    m.mean, m.square = ([fake(k) for k in n] for _ in range(2))
    m.meanCodes, m.rootCodes, m.scales = ([fake(k * b) for b in blocks] for k in (64, 64, 2))
    return m


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw(fake, bits):  # noqa: F811
    for name, values in (("learningRate", (-1e-3, float("nan"), float("inf"))), ("beta1", (-0.1, 1.0, float("nan"))), ("beta2", (-0.1, 1.0, 1.5)),
                         ("epsilon", (0.0, -1e-8, 1e-40, 1e38, float("nan"))), ("weightDecay", (-0.1, float("inf")))):
        for v in values:
            m = adamw(fake, bits)
            setattr(m, name, v)
            with pytest.raises(gt.THCError, match="learning rate|beta1|beta2|epsilon|decay"):
                m.update()
    m = adamw(fake, bits)
    m.step = fake(1)
    with pytest.raises(gt.THCError, match="step of 2 values"):
        m.update()
    kept = ("mean", "square") if bits == 32 else ("meanCodes", "rootCodes", "scales")
    for name in ("gradWeights",) + kept:
        m = adamw(fake, bits)
        n = getattr(m, name)[1].nElement()
        for bad in (fake(n + 1), fake(n, strides=(2,))):
            setattr(m, name, changed(getattr(m, name), 1, bad))
            with pytest.raises(gt.THCError, match="for tensor 2"):
                m.update()
        m = adamw(fake, bits)
        setattr(m, name, getattr(m, name)[:-1])
        with pytest.raises(ValueError):
            m.update()
    m = adamw(fake, bits)
    m.weights = changed(m.weights, 0, fake(7, 3, strides=(1, 7)))
    with pytest.raises(gt.THCError, match="contiguous weights"):
        m.update()
    # the same tensor twice, the end of one in another, a gradient in what is written
    for name, i, other in (("weights", 2, lambda m: m.weights[2]), (kept[0], 1, lambda m: getattr(m, kept[1])[1]), ("gradWeights", 1, lambda m: m.weights[1]),
                           ("gradWeights", 2, lambda m: getattr(m, kept[-1])[2] if bits == 32 else m.weights[2])):
        m = adamw(fake, bits)
        if name == "weights":
            m.weights += (m.weights[2],)
            m.gradWeights += (fake(300),)
            for k in kept:
                setattr(m, k, getattr(m, k) + (fake(getattr(m, k)[2].nElement()),))
        else:
            setattr(m, name, changed(getattr(m, name), i, other(m)))
        with pytest.raises(gt.THCError, match="shares memory"):
            m.update()
    m = adamw(fake, bits)
    m.step = m.weights[1].narrow(1, 255, 2)
    with pytest.raises(gt.THCError, match="shares memory"):
        m.update()
    m = adamw(fake, bits)
    m.gradWeights = changed(m.gradWeights, 0, m.weights[1].narrow(1, 256 - 20, 21))
    with pytest.raises(gt.THCError, match="shares memory"):
        m.update()


def changed(tensors, i, t):
    tensors = list(tensors)
    tensors[i] = t
    return tensors


def test_adamw_arguments(fake):  # noqa: F811
    w = fake(5)
    for args, kw, error in ((([w], [w, w]), {}, ValueError), (([w], [w]), {"bits": 16}, ValueError), ((np.zeros(3), [w]), {}, TypeError)):
        with pytest.raises(error):
            optim.AdamW(*args, **kw)
    m = adamw(fake, 32)
    assert m.moments() == (m.mean, m.square)
    with pytest.raises(ValueError):
        m.moments(m.mean, m.square)
    m = adamw(fake, 8)
    with pytest.raises(ValueError):
        m.moments(m.mean[:2], m.square)
    with pytest.raises(gt.THCError, match="shares memory"):
        m.moments(m.mean, changed(m.square, 1, m.mean[1]))
    m.scales = changed(m.scales, 2, fake(5).narrow(1, 2, 4))
    with pytest.raises(gt.THCError, match="boundary of 8 bytes"):
        m.update()
    with pytest.raises(gt.THCError, match="boundary of 8 bytes"):
        m.moments(m.mean, m.square)


def test_parameters_of_modules():
    """Those of containers' modules too; modules without any add nothing."""
    a, b = nn.Linear(3, 2), nn.LayerNorm(2)
    net = nn.Sequential().add(a).add(nn.Sequential().add(nn.Router(1)).add(b)).add(nn.LayerNorm(2, affine=False))
    weights, gradients = optim.parameters(net, a)
    assert [id(t) for t in weights] == [id(t) for t in (a.weight, a.bias, b.weight, b.bias, a.weight, a.bias)]
    assert [id(t) for t in gradients] == [id(t) for t in (a.gradWeight, a.gradBias, b.gradWeight, b.gradBias, a.gradWeight, a.gradBias)]
    with pytest.raises(TypeError, match="call :gpu"):
        optim.AdamW(*optim.parameters(net))


def test_adamw_keeps_the_tensors_it_is_given(fake):  # noqa: F811
    """What the library gets are the tensors of the fields, also after others have been put there; a field is no list to be changed behind it."""
    m = adamw(fake)
    with pytest.raises(TypeError):
        m.mean[1] = fake(256)
    with pytest.raises(TypeError):
        m.mean = [fake(256), np.zeros(3)]
    m.mean = [fake(7, 3), fake(256), fake(300)]
    array = m._arrays("mean")[0]
    assert [C.addressof(array[i].contents) for i in range(3)] == [C.addressof(t._p.contents) for t in m.mean]
    state = m.__getstate__()
    assert state["_lists"]["mean"] is m.mean
    twin = object.__new__(optim.AdamW)
    twin.__setstate__(state)
    assert twin.mean == m.mean and twin.beta1 == m.beta1


def test_tensors_of_another_device(fake):  # noqa: F811
    m = router(fake)
    with pytest.raises(gt.THCError, match="Invalid argument 1: tensor of device 2"):
        m.forward(fake(5, 6, device=2))
    m = dispatch(fake)
    with pytest.raises(gt.THCError, match="Invalid argument 2: tensor of device 2"):
        m.forward([fake(5, 6), fake(5, 2, device=2)])
    m = combine(fake)
    with pytest.raises(gt.THCError, match="Invalid argument 4: tensor of device 2"):
        m.forward([fake(8, 6), fake(5, 2), fake(5, 2), fake(5, 6, device=2)])
    m = adamw(fake)
    m.square = changed(m.square, 2, fake(300, device=2))
    with pytest.raises(gt.THCError, match="Invalid argument 5: tensor of device 2"):
        m.update()


def test_missing_tensors():
    L = gt.lib()
    counts, none = np.zeros(2, np.int64), (TP * 1)()
    for call in (lambda: L.THGPUNN_Router_updateOutput(None, None, None, 1, 1), lambda: L.THGPUNN_Router_updateGradInput(None, None, None, None, None, 1),
                 lambda: L.THGPUNN_Dispatch_updateOutput(None, None, None, None, counts, 2), lambda: L.THGPUNN_Dispatch_updateGradInput(None, None, None, None),
                 lambda: L.THGPUNN_Combine_updateOutput(None, None, None, None, None, 4), lambda: L.THGPUNN_Combine_backward(None, None, None, None, None, None)):
        with pytest.raises(gt.THCError, match="tensors expected"):
            call()
    with pytest.raises(gt.THCError, match="Invalid argument 6: tensors expected"):
        L.THGPUNN_AdamW_update(1, none, none, none, none, None, 1e-3, 0.9, 0.999, 1e-8, 0.0)
    for array in (none, C.cast(none, C.POINTER(TP))):      # an array, or a pointer to its first
        with pytest.raises(gt.THCError, match="tensors expected"):
            L.THGPUNN_AdamW8_moments(1, array, array, array, array, array)
    for bad in (5, (C.c_long * 2)(), [None]):
        with pytest.raises((C.ArgumentError, TypeError)):
            L.THGPUNN_AdamW8_moments(1, bad, none, none, none, none)
