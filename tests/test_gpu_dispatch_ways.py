"""nn.Dispatch: each block of the copy ranks the slots for itself only where that reads little, which shows in the number of launches; the results are the same on both sides."""
import numpy as np
import pytest

from test_gpu_dispatch import experts_of, f32, normal, plan

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gt():
    import mcw_cppamp_torch_b200 as gt
    return gt


# tokens, slots of each, values of a row, launches: every block reads all slots in one launch, or one before the copy ranks them
@pytest.mark.parametrize("tokens,k,size,launches", [(24, 8, 4096, 1), (1, 1, 1, 1), (256, 8, 1024, 1), (1024, 1, 1024, 1), (1025, 1, 1024, 2), (512, 1, 4096, 1), (513, 1, 4096, 2),
                                                    (2048, 1, 16, 2), (2048, 1, 4095, 2), (512, 2, 512, 1), (512, 2, 511, 1), (513, 2, 511, 2), (128, 8, 1025, 1), (128, 8, 4095, 2), (2, 64, 2000, 1),
                                                    (2, 65, 2000, 2)])
def test_few_slots_by_what_blocks_read(gt, tokens, k, size, launches):
    x, e = normal(tokens, tokens, size), experts_of(size, tokens, k, 37)
    order, places, counts = plan(e, 37)
    m, input = gt.nn.Dispatch(37), [gt.gpu(x), gt.gpu(f32(e))]
    before = gt.lib().THGPUKernelLaunchCount()
    rows, told = m.forward(input)
    assert gt.lib().THGPUKernelLaunchCount() - before == launches
    assert np.array_equal(rows.float(), x[order // k] if order.size else np.zeros(0)) and np.array_equal(told, counts) and np.array_equal(m.positions.float(), places)
