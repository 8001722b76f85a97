"""nn.GroupedLinear where one group has most of the rows: results, and the device memory that a call takes for itself."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch

from test_gpu_feedforward import wrap
from test_gpu_fused_linear import check_groups, down, gt, randn, up  # noqa: F401

pytestmark = pytest.mark.gpu


def uneven(n, few, long):
    """n groups of `few` rows, but for those that `long` names: place -> rows."""
    counts = [few] * n
    for at, rows in long.items():
        counts[at] = rows
    return counts


@pytest.mark.parametrize("counts", [uneven(40, 18, {17: 5000}), uneven(6, 0, {0: 3001}), uneven(30, 20, {29: 1025}), uneven(30, 33, {3: 2048, 4: 2049, 21: 700}),
                                    uneven(200, 17, {0: 9000, 199: 4100}), uneven(3, 513, {})])
@pytest.mark.parametrize("I,O", [(64, 64), (33, 131), (130, 7), (1, 20), (260, 16)])
def test_results(gt, counts, I, O):  # noqa: F811
    """Weight gradients cut along k for some groups and not for others, the long ones first, last and between."""
    check_groups(gt, counts, I, O, "none")


MEMORY = """
import numpy as np, torch, mcw_cppamp_torch_b200 as gt
groups, few, longest, width, out = %r
counts = np.full(groups, few); counts[groups // 3] = longest
rows = int(counts.sum())
m = gt.nn.GroupedLinear(groups, width, out).gpu()
x, g = gt.GPUTensor(rows, width).fill(1.0), gt.GPUTensor(rows, out).fill(0.5)
m.zeroGradParameters()
few = gt.nn.GroupedLinear(2, width, out).gpu()
few.accGradParameters([x.narrow(1, 1, 40), [20, 20]], g.narrow(1, 1, 40))       # (the first scratch there is)
gt.synchronize()
before = torch.cuda.mem_get_info()[0]
m.accGradParameters([x, counts], g)
gt.synchronize()
took = before - torch.cuda.mem_get_info()[0]
assert torch.equal(torch.from_numpy(m.gradWeight.float()), torch.from_numpy(0.5 * counts.astype(np.float32))[:, None, None].expand(groups, out, width))
print("took", took)
"""


@pytest.mark.parametrize("sizes", [(128, 20, 13800, 256, 256), (1000, 20, 13800, 128, 128), (2048, 17, 16384, 64, 64)])
def test_scratch_of_weight_gradients(sizes):
    """What a call takes in all: partial sums of fewer than six tiles of 16 KB an SM and bias gradients' parts, in steps of 64 MB of the arena, which grows
    by half at least: 128 MB at most.  A gradient of 34 to 66 MB once took 0.7 to 1.8 GB here."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", MEMORY % (sizes,)], cwd=root, env=dict(os.environ, PYTHONPATH=root), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    assert int(r.stdout.split()[-1]) <= 128 << 20


def test_recorded_and_replayed(gt):  # noqa: F811
    """Tickets and partial sums of cut groups inside a recording, with calls of other counts between its runs."""
    counts, others = uneven(30, 18, {3: 5000, 20: 1500}), uneven(30, 600, {29: 9})
    rows, more = sum(counts), sum(others)
    m = gt.nn.GroupedLinear(30, 70, 90).gpu()
    x, g = torch.zeros(rows, 70, device="cuda"), torch.zeros(rows, 90, device="cuda")
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    gt.lib().THGPUSetStream(ctypes.c_void_p(stream.cuda_stream))
    try:
        X, G, X2, G2 = wrap(gt, x), wrap(gt, g), up(gt, randn(5, more, 70)), up(gt, randn(6, more, 90))

        def step():
            m.gradWeight.fill(0.25)
            m.accGradParameters([X, counts], G)
        for _ in range(2):
            step()
        gt.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for seed in (1, 2, 3):
            x.copy_(randn(seed, rows, 70)); g.copy_(randn(seed + 10, rows, 90))
            torch.cuda.synchronize()
            step()
            gt.synchronize()
            want = down(m.gradWeight).clone()
            m.accGradParameters([X2, others], G2)
            gt.synchronize()
            with torch.cuda.stream(stream):
                graph.replay()
            gt.synchronize()
            assert torch.equal(down(m.gradWeight), want)
        del graph
    finally:
        gt.synchronize()
        gt.lib().THGPUSetStream(None)
