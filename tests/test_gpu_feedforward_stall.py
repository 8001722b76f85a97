"""Products of few rows behind a kernel whose bounded wait has run out: as all products, they leave their results alone.  What runs out here is the wait of the
one-warp probe that tests/test_gpu_stall.py has."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gt():
    import mcw_cppamp_torch_b200 as m
    m.lib().THGPUInit()
    return m


# rows of a group, groups, inputs, outputs: the pieces of gradInput summed in one block, and in several that meet by tickets
@pytest.mark.parametrize("rows,groups,inputs,outputs", [(7, 1, 40, 24), (3, 1, 130, 33), (1, 8, 24, 40), (8, 9, 130, 700), (2, 12, 333, 2049)])
def test_gradients_of_few_rows(gt, rows, groups, inputs, outputs):
    L = gt.lib()
    n = rows * groups
    counts = np.full(groups, rows, np.int64)
    x, g = gt.GPUTensor(n, inputs).fill(1.0), gt.GPUTensor(n, outputs).fill(1.0)
    shape = (groups, outputs, inputs) if groups > 1 else (outputs, inputs)
    w, gw, gi = gt.GPUTensor(*shape).fill(0.5), gt.GPUTensor(*shape), gt.GPUTensor(n, inputs)

    def backward():
        if groups > 1:
            L.THGPUNN_GroupedLinear_backward(x._p, counts, groups, g._p, gi._p, None, None, w._p, gw._p, None, 0, 1.0)
        else:
            L.THGPUNN_FusedLinear_backward(x._p, g._p, gi._p, None, None, w._p, gw._p, None, 0, 1.0)

    for _ in range(2):
        gw.fill(0.25)
        gi.fill(-1)
        L.THGPUSynchronize()
        L.THGPUStallProbe(2048)
        backward()
        with pytest.raises(gt.THCError, match="pipeline stall"):
            L.THGPUSynchronize()
        assert (gw.float() == 0.25).all()
        assert (gi.float() == -1).all()
        backward()                                   # the flag is cleared, the tickets are as they were
        assert (gw.float() == 0.25 + rows).all()
        assert (gi.float() == 0.5 * outputs).all()
