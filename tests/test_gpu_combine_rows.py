"""nn.Combine where some rows have no slot, as when slots are dropped behind nn.Dispatch: their gradient is zero, whatever lay there."""
import ctypes

import numpy as np
import pytest
import torch

from test_gpu_dispatch import U, exact_combine, experts_of, f32, normal, plan

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gt():
    import mcw_cppamp_torch_b200 as gt
    return gt


def dropped(seed, tokens, k, groups, share):
    """Places as Dispatch leaves them, some of them set to 0 behind it, and the number of rows."""
    places = plan(experts_of(seed, tokens, k, groups, 0.1), groups)[1]
    n = int(places.max())
    places[np.random.RandomState(seed + 1).random_sample(places.shape) < share] = 0
    return places, n


# few rows and many, by which rows without a slot are looked for in pieces or all are cleared; rows that 16 bytes divide and others
CASES = [(2, 1, 3, 4), (24, 8, 64, 4096), (100, 3, 7, 333), (40, 70, 9, 40), (513, 4, 37, 64), (2100, 3, 9, 1023), (8192, 4, 9, 5), (8193, 4, 9, 5), (6000, 8, 130, 72),
         (17000, 2, 5, 128), (70000, 1, 3, 96), (40000, 3, 11, 20), (33000, 1, 5, 1)]


@pytest.mark.parametrize("tokens,k,groups,size", CASES)
@pytest.mark.parametrize("share", [0.02, 0.5, 1.0])
def test_rows_without_a_slot(gt, tokens, k, groups, size, share):
    places, n = dropped(size, tokens, k, groups, share)
    z, w, g = normal(1, n, size), normal(2, tokens, k), normal(4, tokens, size)
    y, mass, gz, gw, wmass = exact_combine(z, w, places, None, g)
    room = gt.GPUTensor(n + 3, size).fill(np.nan)
    m = gt.nn.Combine()
    m.gradRows = room.narrow(1, 1, n)
    input = [gt.gpu(z), gt.gpu(w), gt.gpu(f32(places))]
    assert np.all(np.abs(m.forward(input).float() - y) <= (k + 1) * U * mass)
    G = gt.gpu(g)
    back = m.backward(input, G)
    got = back[0].float()
    assert np.all(np.abs(got - gz) <= U * np.abs(gz))              # (NaN would compare false)
    named = np.zeros(n, bool)
    named[places[places > 0] - 1] = True
    assert not got[~named].any() and np.isnan(room.float()[n:]).all()
    assert np.all(np.abs(back[1].float() - gw) <= (size / 32 + 10) * U * wmass)
    # the rows' gradient alone, without weights, at another address
    flat = gt.GPUTensor(n * size + 1).fill(np.nan)
    alone = flat.narrow(1, 2, n * size).view(n, size)
    gt.lib().THGPUNN_Combine_backward(input[0]._p, None, input[2]._p, G._p, alone._p, None)
    ones = exact_combine(z, np.ones((tokens, k), np.float32), places, None, g)[2]
    assert np.array_equal(alone.float(), ones.astype(np.float32)) and np.isnan(flat.float()[0])


def test_places_outside_the_rows_name_none(gt):
    z, w, g = normal(1, 6, 20), normal(2, 4, 3), normal(4, 4, 20)
    places = np.array([[1, 7, 0], [3, np.nan, -2], [np.inf, 0.5, 1e30], [0, 5, 0]], np.float32)
    m = gt.nn.Combine()
    m.gradRows = gt.GPUTensor(6, 20).fill(np.nan)
    back = m.backward([gt.gpu(z), gt.gpu(w), gt.gpu(places)], gt.gpu(g))[0].float()
    assert not back[[1, 3, 5]].any() and back[[0, 2, 4]].all()


def test_more_rows_than_places_can_name(gt):
    n = 2 ** 24 + 40001
    z, places = gt.GPUTensor(n, 1).fill(1.0), np.array([[2 ** 24, 1], [0, 2 ** 24 - 1], [2 ** 24 + 2, 32769]], np.float32)
    m = gt.nn.Combine()
    m.gradRows = gt.GPUTensor(n, 1).fill(np.nan)
    g = gt.gpu(np.full((3, 1), 2.0, np.float32))
    back = m.backward([z, None, gt.gpu(places)], g)[0].float()
    want = np.zeros((n, 1), np.float32)
    want[[2 ** 24 - 1, 0, 2 ** 24 - 2, 32768]] = 2
    assert np.array_equal(back, want)


def test_no_tokens(gt):
    """Rows, and no token that has one of them."""
    m = gt.nn.Combine(20)
    m.gradRows = gt.GPUTensor(6, 20).fill(np.nan)
    empty = gt.GPUTensor()
    back = m.backward([gt.gpu(normal(1, 6, 20)), gt.GPUTensor(), empty], empty)[0]
    assert back.size() == (6, 20) and not back.float().any()


def test_recorded_and_replayed(gt):
    """Other slots dropped at each replay, in pieces and cleared as a whole."""
    stream = torch.cuda.Stream()
    gt.synchronize()
    gt.lib().THGPUSetStream(ctypes.c_void_p(stream.cuda_stream))
    try:
        for tokens, k, size in ((300, 3, 100), (12000, 3, 9)):
            places = plan(experts_of(1, tokens, k, 6, 0.0), 6)[1]
            n = int(places.max())
            z, w, g = normal(1, n, size), normal(2, tokens, k), normal(4, tokens, size)
            P, m = gt.gpu(f32(places)), gt.nn.Combine()
            input, G = [gt.gpu(z), gt.gpu(w), P], gt.gpu(g)
            m.backward(input, G)
            gt.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                m.backward(input, G)
            for seed in range(3):
                now = np.where(np.random.RandomState(seed).random_sample(places.shape) < 0.3, 0, places)
                P.copy(f32(now))
                m.gradRows.fill(np.nan)
                gt.synchronize()
                with torch.cuda.stream(stream):
                    graph.replay()
                gt.synchronize()
                gz = exact_combine(z, w, now, None, g)[2]
                assert np.all(np.abs(m.gradRows.float() - gz) <= U * np.abs(gz))
            del graph
    finally:
        gt.synchronize()
        gt.lib().THGPUSetStream(None)
