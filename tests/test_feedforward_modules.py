"""What the modules LayerNorm, FusedLinear and GroupedLinear do on the host around their library calls.  Tensors are shapes over memory that nothing reads,
as in tests/test_feedforward_refusals.py, but for the tests that are marked."""
import numpy as np
import pytest

import mcw_cppamp_torch_b200 as gt
from mcw_cppamp_torch_b200 import nn
from test_feedforward_refusals import fake, grouped, linear, norm  # noqa: F401


@pytest.mark.parametrize("sizes,shape", [((6, 5), (4, 5, 6)), ((6, 5), (5, 6)), ((6, 5), (4, 3, 10)), ((4, 6, 5), (2, 4, 5, 6)), ((4, 6, 5), (6, 4, 5)),
                                         ((2, 8), (3, 4, 4)), ((3, 4), (4, 1, 3))])
def test_layer_norm_refuses_other_sizes_of_the_same_product(fake, sizes, shape):  # noqa: F811
    m = norm(fake, sizes[0])
    m.__init__(*sizes)
    m.weight, m.bias = fake(m.size), fake(m.size)
    with pytest.raises(ValueError, match="trailing sizes"):
        m.forward(fake(*shape))


@pytest.mark.parametrize("sizes,shape", [((6, 5), (4, 6, 5)), ((6, 5), (6, 5)), ((6, 5), (7, 30)), ((6, 5), (30,)), ((6, 5), (3, 2, 3, 5)), ((30,), (4, 5, 6)),
                                         ((30,), (4, 30)), ((4, 6, 5), (3, 24, 5)), ((4, 6, 5), (4, 30)), ((6, 1, 5), (6, 5)), ((6, 5), (6, 1, 5)), ((1, 1), (4, 3)),
                                         ((6, 5), (6, 5, 1)), ((1, 6, 5), (2, 6, 5))])
def test_layer_norm_takes_merged_and_split_sizes(fake, monkeypatch, sizes, shape):  # noqa: F811
    calls = []

    class Library:
        def THGPUNN_LayerNorm_updateOutput(self, *args):
            calls.append(args)
    m = nn.LayerNorm(*sizes)
    m.weight, m.bias = fake(m.size), fake(m.size)
    x = fake(*shape)
    monkeypatch.setattr(nn, "lib", Library)
    m.forward(x)
    assert len(calls) == 1 and calls[0][6] == m.size


def test_layer_norm_refuses_sizes_that_make_no_row(fake):  # noqa: F811
    m = nn.LayerNorm(6, 5)
    m.weight, m.bias = fake(30), fake(30)
    with pytest.raises(ValueError, match="trailing sizes"):
        m.forward(fake(4, 7))


@pytest.mark.parametrize("make,bad", [(norm, lambda f: f(5, 9)), (linear, lambda f: f(5, 7)), (grouped, lambda f: [f(5, 7), [2, 0, 3]])])
@pytest.mark.parametrize("kept", [True, False])
def test_a_refused_forward_pass_changes_nothing_about_what_is_kept(fake, make, bad, kept):  # noqa: F811
    """Behind an evaluation, a training pass that is refused leaves the module with nothing to go back by; and one that evaluates leaves what there was."""
    m = make(fake)
    m._kept, m.train = kept, not kept
    with pytest.raises(gt.THCError):
        m.forward(bad(fake))
    assert m._kept is kept


def test_the_callers_gradient_is_not_saved(fake):  # noqa: F811
    m, rows = linear(fake), fake(5, 6)
    for gradInput, want in (([rows, fake(5, 4)], rows), (rows, rows), (None, None)):
        m.gradInput = gradInput
        state = m.__getstate__()
        assert state["gradInput"] is want and m.gradInput is gradInput and set(state) == set(m.__dict__)


@pytest.mark.gpu
def test_a_clone_behind_a_call_with_a_residual():
    m = nn.FusedLinear(6, 4, "gelu").gpu()
    rs = np.random.RandomState(0)
    x, r, g = (gt.gpu(rs.randn(5, n).astype(np.float32)) for n in (6, 4, 4))
    m.zeroGradParameters()
    m.forward([x, r])
    rows = m.backward([x, r], g)[0].float()
    twin = m.clone()
    assert isinstance(twin.gradInput, gt.GPUTensor) and np.array_equal(twin.gradInput.float(), rows)
    assert np.array_equal(twin.forward([x, r]).float(), m.output.float())
    first, second = twin.backward([x, r], g)
    assert second is g and np.array_equal(first.float(), rows)
