"""What LayerNorm, FusedLinear and GroupedLinear refuse, before any device is touched: tensors here are shapes over memory that nothing reads."""
import ctypes as C

import numpy as np
import pytest

import mcw_cppamp_torch_b200 as gt
from mcw_cppamp_torch_b200 import nn


class Fake:
    """Tensors at addresses of their own, far apart."""

    def __init__(self):
        self.next = 1 << 32

    def __call__(self, *sizes, strides=None, at=None, device=0):
        L = gt.lib()
        n = 1 << 20
        base = at or self.next
        self.next += 1 << 24
        st = L.THGPUStorage_newWithData(C.c_void_p(base), n)
        st.contents.allocatorContext = device
        t = gt.GPUTensor(_ptr=L.THGPUTensor_newWithStorage1d(st, 0, n, 1))
        L.THGPUStorage_free(st)
        size = (C.c_long * len(sizes))(*sizes)
        from mcw_cppamp_torch_b200.tensor import _long_storage
        L.THGPUTensor_setStorage(t._p, t._p.contents.storage, 0, C.byref(_long_storage(list(sizes))),
                                 C.byref(_long_storage(list(strides))) if strides else None)
        del size
        return t


@pytest.fixture
def fake():
    return Fake()


def norm(fake, size=8):
    m = nn.LayerNorm(size)
    m.weight, m.bias, m.gradWeight, m.gradBias = (fake(size) for _ in range(4))
    m.output, m.gradInput, m.mean, m.invStd = fake(5, size), fake(5, size), fake(5), fake(5)
    return m


def test_layer_norm(fake):
    x, g = fake(5, 8), fake(5, 8)
    for kw in (dict(sizes=()), dict(sizes=(0,)), dict(sizes=(4, 0))):
        with pytest.raises(ValueError):
            nn.LayerNorm(*kw["sizes"])
    with pytest.raises(TypeError):
        norm(fake).forward(np.zeros((5, 8), np.float32))
    with pytest.raises(TypeError):
        nn.LayerNorm(8).forward(x)                                   # parameters still on the host
    m = norm(fake)
    with pytest.raises(gt.THCError, match="trailing dimensions"):
        m.forward(fake(5, 9))
    with pytest.raises(gt.THCError, match="trailing dimensions"):
        m.forward(fake(16, 4, 3))
    for name, bad in (("weight", fake(9)), ("bias", fake(7)), ("weight", fake(8, strides=(2,)))):
        m = norm(fake)
        setattr(m, name, bad)
        with pytest.raises(gt.THCError, match="Invalid argument [34]"):
            m.forward(x)
    m = norm(fake)
    m.eps = -1.0
    with pytest.raises(gt.THCError, match="eps"):
        m.forward(x)
    for name, bad, match in (("output", x, "shares memory"), ("output", fake(5, 8, strides=(9, 1)), "contiguous result"), ("mean", fake(5, strides=(2,)), "contiguous"),
                             ("mean", x.narrow(2, 1, 1).narrow(1, 1, 1), "shares|resiz|no CUDA")):
        m = norm(fake)
        setattr(m, name, bad)
        with pytest.raises(gt.THCError, match=match):
            m.forward(x)
    with pytest.raises(gt.THCError, match="gradOutput"):
        norm(fake).backward(x, fake(5, 7))
    for name, bad, match in (("mean", fake(4), "statistics"), ("invStd", fake(6), "statistics"), ("gradWeight", fake(9), "gradWeight"), ("gradBias", fake(9), "gradBias"),
                             ("gradInput", x, "shares memory"), ("gradInput", g, "shares memory")):
        m = norm(fake)
        setattr(m, name, bad)
        with pytest.raises(gt.THCError, match=match):
            m.backward(x, g)
    L = gt.lib()
    m = norm(fake)
    with pytest.raises(gt.THCError, match="both or neither of weight"):
        L.THGPUNN_LayerNorm_updateOutput(x._p, m.output._p, m.weight._p, None, None, None, 8, 1e-5)
    with pytest.raises(gt.THCError, match="both or neither of mean"):
        L.THGPUNN_LayerNorm_updateOutput(x._p, m.output._p, None, None, m.mean._p, None, 8, 1e-5)
    with pytest.raises(gt.THCError, match="size must be positive"):
        L.THGPUNN_LayerNorm_updateOutput(x._p, m.output._p, None, None, None, None, 0, 1e-5)
    with pytest.raises(gt.THCError, match="both or neither of gradWeight"):
        L.THGPUNN_LayerNorm_backward(x._p, g._p, None, m.weight._p, m.gradWeight._p, None, m.mean._p, m.invStd._p, 8, 1.0)


def linear(fake, act="gelu"):
    m = nn.FusedLinear(6, 4, act)
    m.weight, m.bias, m.gradWeight, m.gradBias = fake(4, 6), fake(4), fake(4, 6), fake(4)
    m.output, m.preactivation, m.gradPreactivation, m.gradInput = fake(5, 4), fake(5, 4), fake(5, 4), fake(5, 6)
    return m


def test_fused_linear(fake):
    x, g = fake(5, 6), fake(5, 4)
    with pytest.raises(ValueError):
        nn.FusedLinear(6, 4, "tanh")
    with pytest.raises(TypeError):
        nn.FusedLinear(6, 4).forward(x)
    with pytest.raises(TypeError):
        linear(fake).forward([x, np.zeros((5, 4), np.float32)])
    with pytest.raises(gt.THCError, match="input size"):
        linear(fake).forward(fake(5, 7))
    with pytest.raises(gt.THCError, match="input size"):
        linear(fake).forward(fake(6))
    with pytest.raises(gt.THCError, match="residual"):
        linear(fake).forward([x, fake(5, 5)])
    for name, bad, match in (("weight", fake(4, 6, strides=(1, 4)), "matrix"), ("weight", fake(24), "matrix"), ("bias", fake(5), "bias"), ("output", x, None),
                             ("output", fake(5, 4, strides=(1, 5)), "contiguous result"), ("preactivation", fake(5, 4, strides=(1, 5)), "contiguous result")):
        m = linear(fake)
        setattr(m, name, bad)
        with pytest.raises(gt.THCError, match=match):
            m.forward(x)
    r = fake(5, 4)
    for name in ("output", "preactivation"):
        m = linear(fake)
        setattr(m, name, r)
        with pytest.raises(gt.THCError, match="shares memory"):
            m.forward([x, r])
    m = linear(fake)
    m.preactivation = m.output
    with pytest.raises(gt.THCError, match="shares memory"):
        m.forward(x)
    with pytest.raises(gt.THCError, match="gradOutput"):
        linear(fake).backward(x, fake(4, 4))
    for name, bad, match in (("preactivation", fake(4, 4), "kept"), ("gradWeight", fake(4, 5), "gradWeight"), ("gradBias", fake(3), "gradBias"),
                             ("gradInput", fake(5, 6, strides=(1, 5)), "contiguous result"), ("gradPreactivation", g, "shares memory")):
        m = linear(fake)
        setattr(m, name, bad)
        with pytest.raises(gt.THCError, match=match):
            m.backward(x, g)
    m = linear(fake)
    m.gradWeight = m.weight
    with pytest.raises(gt.THCError, match="shares memory"):
        m.backward(x, g)
    for code in (-1, 4):
        m = linear(fake)
        m._code = code
        with pytest.raises(gt.THCError, match="activation must be"):
            m.forward(x)


def grouped(fake, act="gelu"):
    m = nn.GroupedLinear(3, 6, 4, act)
    m.weight, m.bias, m.gradWeight, m.gradBias = fake(3, 4, 6), fake(3, 4), fake(3, 4, 6), fake(3, 4)
    m.output, m.preactivation, m.gradPreactivation, m.gradInput = fake(5, 4), fake(5, 4), fake(5, 4), fake(5, 6)
    return m


def test_grouped_linear(fake):
    x, g, counts = fake(5, 6), fake(5, 4), [2, 0, 3]
    for bad in ([2, 3], [2, 0, 3, 0], [2.0, 0.0, 3.0], [[2, 0, 3]], 5):
        with pytest.raises(ValueError):
            grouped(fake).forward([x, bad])
    with pytest.raises(TypeError):
        grouped(fake).forward([x, fake(3)])
    for bad in ([2, 0, 2], [2, 1, 3], [6, -1, 0], [-1, 3, 3], [2, 2 ** 62, 2 ** 62], [2 ** 63 - 1, 2 ** 63 - 1, 7]):
        with pytest.raises(gt.THCError, match="counts must"):
            grouped(fake).forward([x, bad])
        with pytest.raises(gt.THCError, match="counts must"):
            grouped(fake).backward([x, bad], g)
    with pytest.raises(gt.THCError, match="input size"):
        grouped(fake).forward([fake(5, 7), counts])
    for name, bad, match in (("weight", fake(12, 6), "one matrix a group"), ("weight", fake(2, 4, 6), "one matrix a group"), ("bias", fake(12), "bias"),
                             ("output", x, None)):
        m = grouped(fake)
        setattr(m, name, bad)
        with pytest.raises(gt.THCError, match=match):
            m.forward([x, counts])
    for name, bad, match in (("preactivation", fake(4, 4), "kept"), ("gradWeight", fake(3, 6, 4), "gradWeight"), ("gradBias", fake(12), "gradBias"),
                             ("gradPreactivation", g, "shares memory")):
        m = grouped(fake)
        setattr(m, name, bad)
        with pytest.raises(gt.THCError, match=match):
            m.backward([x, counts], g)
    L = gt.lib()
    m = grouped(fake)
    none = np.zeros(0, np.int64)
    with pytest.raises(gt.THCError, match="a count of rows for each group"):
        L.THGPUNN_GroupedLinear_updateOutput(x._p, none, 0, m.output._p, None, m.weight._p, m.bias._p, 0)
    with pytest.raises((C.ArgumentError, TypeError)):
        L.THGPUNN_GroupedLinear_updateOutput(x._p, np.zeros(3, np.int32), 3, m.output._p, None, m.weight._p, m.bias._p, 0)


def test_tensors_of_another_device(fake):
    """A tensor made on the second device while the first is current."""
    here, there = fake(5, 6, device=1), fake(5, 6, device=2)
    m = linear(fake)
    with pytest.raises(gt.THCError, match="Invalid argument 1: tensor of device 2"):
        m.forward(there)
    m.output = fake(5, 4, device=2)
    with pytest.raises(gt.THCError, match="Invalid argument 3: tensor of device 2"):
        m.forward(here)
    m = norm(fake, 6)
    with pytest.raises(gt.THCError, match="Invalid argument 1: tensor of device 2"):
        m.forward(there)
    m = grouped(fake)
    m.weight = fake(3, 4, 6, device=2)
    with pytest.raises(gt.THCError, match="Invalid argument 6: tensor of device 2"):
        m.forward([here, [2, 0, 3]])


def test_missing_tensors():
    L = gt.lib()
    with pytest.raises(gt.THCError, match="tensors expected"):
        L.THGPUNN_LayerNorm_updateOutput(None, None, None, None, None, None, 4, 1e-5)
    with pytest.raises(gt.THCError, match="tensors expected"):
        L.THGPUNN_LayerNorm_backward(None, None, None, None, None, None, None, None, 4, 1.0)
    with pytest.raises(gt.THCError, match="tensors expected"):
        L.THGPUNN_FusedLinear_updateOutput(None, None, None, None, None, None, 0)
    with pytest.raises(gt.THCError, match="tensors expected"):
        L.THGPUNN_FusedLinear_backward(None, None, None, None, None, None, None, None, 0, 1.0)
    counts = np.zeros(2, np.int64)
    with pytest.raises(gt.THCError, match="tensors expected"):
        L.THGPUNN_GroupedLinear_updateOutput(None, counts, 2, None, None, None, None, 0)
    with pytest.raises(gt.THCError, match="tensors expected"):
        L.THGPUNN_GroupedLinear_backward(None, counts, 2, None, None, None, None, None, None, None, 0, 1.0)


def test_a_backward_pass_behind_an_evaluation(fake):
    """After evaluate() a forward pass keeps nothing, and what an earlier one kept is another input's."""
    for m in (norm(fake), linear(fake), grouped(fake)):
        m._kept = False
        x = fake(5, 8) if isinstance(m, nn.LayerNorm) else [fake(5, 6), [2, 0, 3]] if isinstance(m, nn.GroupedLinear) else fake(5, 6)
        for call in (m.backward, m.updateGradInput, m.accGradParameters):
            with pytest.raises(RuntimeError, match="kept nothing"):
                call(x, fake(5, 8) if isinstance(m, nn.LayerNorm) else fake(5, 4))
