"""nn.Dispatch and nn.Combine against their definitions, exactly where they copy and within the roundings of their sums."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def gt():
    import mcw_cppamp_torch_b200 as gt
    return gt


def normal(seed, *shape):
    return np.random.RandomState(seed).standard_normal(shape).astype(np.float32)


def experts_of(seed, tokens, k, groups, none=0.1):
    r = np.random.RandomState(seed)
    e = r.randint(1, groups + 1, (tokens, k))
    e[r.random_sample(e.shape) < none] = 0
    return e


def plan(e, groups):
    """Slots in the order of their rows, their places from 1, and the counts."""
    flat = e.reshape(-1)
    order = np.argsort(np.where(flat > 0, flat, 1 << 30), kind="stable")[:int((flat > 0).sum())]
    places = np.zeros(flat.size, np.int64)
    places[order] = np.arange(1, order.size + 1)
    return order, places.reshape(e.shape), np.bincount(flat, minlength=groups + 1)[1:]


def f32(a):
    return np.ascontiguousarray(a, np.float32)


# few slots, which each block ranks for itself, on both sides of the line, and many; rows that 16-byte accesses divide and others
CASES = [(1, 1, 1, 1), (1, 8, 64, 4096), (3, 2, 4, 5), (24, 8, 64, 1028), (511, 4, 37, 333), (512, 4, 37, 64), (513, 4, 37, 64), (700, 3, 1, 20), (30, 70, 9, 40), (1, 3000, 7, 16),
         (5000, 1, 4096, 36), (40, 5, 4096, 36), (8192, 4, 9, 5), (32769, 1, 9, 5), (1100, 3, 1024, 7), (1100, 3, 1025, 7), (3000, 8, 256, 129), (20000, 6, 130, 32), (97, 2, 5, 5000), (2500, 2, 300, 1024)]


@pytest.mark.parametrize("tokens,k,groups,size", CASES)
@pytest.mark.parametrize("none", [0.0, 0.3])
def test_dispatch(gt, tokens, k, groups, size, none):
    x, e = normal(tokens, tokens, size), experts_of(size, tokens, k, groups, none)
    order, places, counts = plan(e, groups)
    m = gt.nn.Dispatch(groups)
    rows, told = m.forward([gt.gpu(x), gt.gpu(f32(e))])
    assert told.dtype == np.int64 and np.array_equal(told, counts)
    assert np.array_equal(m.positions.float(), places)
    assert np.array_equal(rows.float(), x[order // k] if order.size else np.zeros(0))
    if not order.size:
        return
    g = normal(7, order.size, size)
    gx = m.backward([gt.gpu(x), gt.gpu(f32(e))], [gt.gpu(g), None])[0].float()
    want, mass = (np.zeros((tokens, size)) for _ in range(2))
    for i in range(k):
        t = np.nonzero(places[:, i])[0]
        want[t] += g[places[t, i] - 1]
        mass[t] += np.abs(g[places[t, i] - 1])
    assert np.all(np.abs(gx - want) <= k * U * mass)


def test_experts_named_twice_and_extremes(gt):
    """A token's slots may name one expert; all slots one; none at all."""
    x = normal(0, 40, 12)
    for e in (np.full((40, 3), 2), np.tile([5, 5, 1], (40, 1)), np.full((40, 3), 5)):
        m = gt.nn.Dispatch(5)
        order, places, counts = plan(e, 5)
        rows, told = m.forward([gt.gpu(x), gt.gpu(f32(e))])
        assert np.array_equal(rows.float(), x[order // 3]) and np.array_equal(told, counts)
    for tokens in (40, 900):
        x, none = normal(0, tokens, 12), np.zeros((tokens, 3), np.float32)
        rows, told = m.forward([gt.gpu(x), gt.gpu(none)])
        assert rows.nElement() == 0 and not told.any() and not m.positions.float().any()
        gx = m.backward([gt.gpu(x), gt.gpu(none)], [gt.GPUTensor(), None])[0]
        assert gx.size() == (tokens, 12) and not gx.float().any()
    rows, told = m.forward([gt.GPUTensor(), gt.GPUTensor()])
    assert rows.nElement() == 0 and m.positions.nElement() == 0 and not told.any()
    assert m.backward([gt.GPUTensor(), gt.GPUTensor()], gt.GPUTensor())[0].nElement() == 0


@pytest.mark.parametrize("size", [2100007, 1 << 21])
def test_long_rows(gt, size):
    """Rows of more pieces than a grid's second dimension has blocks, were they as short as those of short rows."""
    x, e = normal(1, 2, size), np.array([[2, 1], [0, 2]])
    order, places, counts = plan(e, 2)
    m = gt.nn.Dispatch(2)
    rows, told = m.forward([gt.gpu(x), gt.gpu(f32(e))])
    assert np.array_equal(rows.float(), x[order // 2]) and np.array_equal(told, counts)
    assert np.array_equal(m.backward([gt.gpu(x), gt.gpu(f32(e))], rows)[0].float(), x * np.array([[2], [1]], np.float32))
    w = np.array([[0.5, 2], [3, -1]], np.float32)
    c = gt.nn.Combine()
    input = [rows, gt.gpu(w), m.positions]
    assert np.array_equal(c.forward(input).float(), x * np.array([[2.5], [-1]], np.float32))
    back = c.backward(input, gt.gpu(x))
    assert np.array_equal(back[0].float(), (w.reshape(-1, 1) * np.repeat(x, 2, 0))[order])
    dot = (x.astype(np.float64) ** 2).sum(1)
    assert np.all(np.abs(back[1].float() - (e > 0) * dot[:, None]) <= (size / 32 + 10) * U * dot[:, None])


@pytest.mark.parametrize("tokens", [50, 3000])
@pytest.mark.parametrize("bad", [0.5, -1.0, 10.0, np.nan, np.inf, -np.inf, 1e30, -0.5])
def test_numbers_that_are_no_experts(gt, tokens, bad):
    """An error, with the number of slots, after work that takes them as none; the next call is as ever."""
    x, e = normal(1, tokens, 8), f32(experts_of(2, tokens, 2, 9))
    e[7, 1] = e[tokens - 1, 0] = bad
    m = gt.nn.Dispatch(9)
    with pytest.raises(gt.THCError, match="Invalid argument 2: 2 slots"):
        m.forward([gt.gpu(x), gt.gpu(e)])
    e[7, 1] = e[tokens - 1, 0] = 0
    order, places, counts = plan(e.astype(np.int64), 9)
    assert np.array_equal(m.positions.float(), places)
    rows, told = m.forward([gt.gpu(x), gt.gpu(e)])
    assert np.array_equal(rows.float(), x[order // 2]) and np.array_equal(told, counts)
    e[7, 1] = -0.0
    assert np.array_equal(m.forward([gt.gpu(x), gt.gpu(e)])[1], counts)


@pytest.mark.parametrize("tokens", [30, 1500])
def test_memory_behind_the_rows_stays(gt, tokens):
    e = experts_of(3, tokens, 2, 6, 0.4)
    order, places, counts = plan(e, 6)
    x = normal(1, tokens, 16)
    m = gt.nn.Dispatch(6)
    room = gt.GPUTensor(tokens * 2 + 5, 16).fill(7.0)
    m.rows = room.narrow(1, 1, tokens * 2)
    rows = m.forward([gt.gpu(x), gt.gpu(f32(e))])[0]
    assert np.array_equal(rows.float(), x[order // 2]) and rows.data_ptr() == room.data_ptr()
    assert np.all(room.float()[order.size:] == 7.0)


@pytest.mark.parametrize("tokens,k", [(90, 3), (1100, 3), (1366, 3), (13000, 3)])
def test_numbers_at_any_address(gt, tokens, k):
    """Expert numbers that start one value behind a 16-byte boundary, as part of a larger storage; none in the last rows."""
    x, e = normal(1, tokens, 6), experts_of(2, tokens, k, 50)
    e[tokens - 7:] = 0
    order, places, counts = plan(e, 50)
    for off in (1, 2, 3):
        room = gt.GPUTensor(tokens * k + 8).fill(-1.0)
        E = room.narrow(1, 1 + off, tokens * k).view(tokens, k)
        E.copy(f32(e))
        m = gt.nn.Dispatch(50)
        rows, told = m.forward([gt.gpu(x), E])
        assert np.array_equal(rows.float(), x[order // k]) and np.array_equal(told, counts) and np.array_equal(m.positions.float(), places)


def test_rows_apart_and_transposed(gt):
    e = experts_of(3, 600, 4, 6)
    order, places, counts = plan(e, 6)
    for size in (64, 63):
        x = normal(1, 600, size)
        wide = gt.GPUTensor(600, size + 9).fill(np.nan)
        v = wide.narrow(2, 6, size)
        v.copy(gt.gpu(x))
        et = gt.gpu(np.ascontiguousarray(f32(e).T)).t()
        for t in (v, gt.gpu(np.ascontiguousarray(x.T)).t()):
            m = gt.nn.Dispatch(6)
            assert np.array_equal(m.forward([t, et])[0].float(), x[order // 4])
            g = gt.GPUTensor(order.size, size + 3).fill(1.0).narrow(2, 2, size)
            gx = m.backward([t, et], g)[0].float()
            assert np.array_equal(gx, np.repeat((e > 0).sum(1)[:, None], size, 1))


# ------------------------------------------------------------------ Combine
def exact_combine(z, w, places, r, g):
    z, w, g = z.astype(np.float64), w.astype(np.float64), g.astype(np.float64)
    tokens, size = g.shape
    y, mass = (np.zeros((tokens, size)) if r is None else r.astype(np.float64) for _ in range(2))
    y, mass = y.copy(), np.abs(mass)
    gz, gw, wmass = np.zeros(z.shape), np.zeros(w.shape), np.zeros(w.shape)
    for i in range(w.shape[1]):
        t = np.nonzero(places[:, i])[0]
        rows = places[t, i] - 1
        y[t] += w[t, i][:, None] * z[rows]
        mass[t] += np.abs(w[t, i][:, None] * z[rows])
        gz[rows] = w[t, i][:, None] * g[t]
        gw[t, i] = (g[t] * z[rows]).sum(1)
        wmass[t, i] = np.abs(g[t] * z[rows]).sum(1)
    return y, mass, gz, gw, wmass


@pytest.mark.parametrize("tokens,k,groups,size", [c for c in CASES if c[1] < 3000 or c[3] <= 16] + [(40, 40, 9, 200), (6, 3, 4, 8200), (5, 33, 2, 9001), (3, 2, 4, 4097)])
@pytest.mark.parametrize("residual,weighted", [(False, True), (True, True), (True, False), (False, False)])
def test_combine(gt, tokens, k, groups, size, residual, weighted):
    places = plan(experts_of(size, tokens, k, groups, 0.2), groups)[1]
    if not places.any():
        places[0, 0] = 1
    n = int(places.max())
    z, w, g = normal(1, n, size), normal(2, tokens, k) if weighted else np.ones((tokens, k), np.float32), normal(4, tokens, size)
    r = normal(3, tokens, size) if residual else None
    y, mass, gz, gw, wmass = exact_combine(z, w, places, r, g)
    given = w.copy()
    given[places == 0] = np.nan                               # weights of slots without a row are not looked at
    m = gt.nn.Combine()
    input = [gt.gpu(z), gt.gpu(given) if weighted else None, gt.gpu(f32(places))] + ([gt.gpu(r)] if residual else [])
    assert np.all(np.abs(m.forward(input).float() - y) <= (k + 1) * U * mass)
    grad = gt.gpu(g)
    back = m.backward(input, grad)
    assert len(back) == 3 + residual and back[2] is None and (not residual or back[3] is grad)
    assert np.all(np.abs(back[0].float() - gz) <= U * np.abs(gz))
    if not weighted:
        assert back[1] is None
        return
    # a thread sums at most ceil(size / 32) products, 5 + 3 additions join the threads
    assert np.all(np.abs(back[1].float() - gw) <= (size / 32 + 10) * U * wmass)
    assert not back[1].float()[places == 0].any()


def test_combine_parts_of_the_gradient(gt):
    """Either gradient alone, through the C functions, is what both together are."""
    places = plan(experts_of(1, 50, 3, 4), 4)[1]
    n = int(places.max())
    z, w, p, g = gt.gpu(normal(1, n, 100)), gt.gpu(normal(2, 50, 3)), gt.gpu(f32(places)), gt.gpu(normal(4, 50, 100))
    m = gt.nn.Combine()
    both = [t.float() for t in m.backward([z, w, p], g)[:2]]
    a, b, L = gt.GPUTensor(), gt.GPUTensor(), gt.lib()
    L.THGPUNN_Combine_backward(z._p, w._p, p._p, g._p, a._p, None)
    L.THGPUNN_Combine_backward(z._p, w._p, p._p, g._p, None, b._p)
    assert np.array_equal(a.float(), both[0]) and np.array_equal(b.float(), both[1])
    L.THGPUNN_Combine_backward(z._p, w._p, p._p, g._p, None, None)


def test_places_of_no_row(gt):
    """Places that are none of the rows' are passed over, and nothing behind the rows is touched."""
    z, w, g = normal(1, 6, 20), normal(2, 4, 3), normal(4, 4, 20)
    places = np.array([[1, 7, 2], [3, np.nan, -2], [np.inf, 4, 1e30], [0, 5, 6]], np.float32)
    good = np.where(np.isin(places, np.arange(1, 7)), places, 0).astype(np.int64)
    y, mass, gz, gw, wmass = exact_combine(z, w, good, None, g)
    m = gt.nn.Combine()
    room = gt.GPUTensor(9, 20).fill(7.0)
    m.gradRows = room.narrow(1, 1, 6)
    input = [gt.gpu(z), gt.gpu(w), gt.gpu(places)]
    assert np.all(np.abs(m.forward(input).float() - y) <= 4 * U * mass)
    big = 2.0 ** 24 + 4                                        # beyond what a float counts: of more rows than that, too
    many = gt.GPUTensor(2 ** 24 + 3, 1).fill(1.0)
    assert not gt.nn.Combine().forward([many, None, gt.gpu(np.full((3, 2), big, np.float32))]).float().any()
    m.backward(input, gt.gpu(g))
    assert np.all(np.abs(room.float()[:6] - gz) <= U * np.abs(gz)) and np.all(room.float()[6:] == 7.0)
    assert np.all(np.abs(m.gradWeights.float() - gw) <= 12 * U * wmass)


def test_combine_without_rows(gt):
    """All tokens behind the last sequence: the residual, or zeros of a given size."""
    none, w, r, g = gt.gpu(np.zeros((5, 2), np.float32)), gt.gpu(normal(2, 5, 2)), normal(3, 5, 24), gt.gpu(normal(4, 5, 24))
    m = gt.nn.Combine()
    assert np.array_equal(m.forward([gt.GPUTensor(), w, none, gt.gpu(r)]).float(), r)
    back = m.backward([gt.GPUTensor(), w, none, gt.gpu(r)], g)
    assert back[0].nElement() == 0 and back[1].size() == (5, 2) and not back[1].float().any()
    m = gt.nn.Combine(24)
    assert m.forward([gt.GPUTensor(), w, none]).size() == (5, 24) and not m.output.float().any()
    assert gt.nn.Combine().forward([gt.GPUTensor(), gt.GPUTensor(), gt.GPUTensor()]).nElement() == 0


def test_combine_strides(gt):
    places = plan(experts_of(1, 50, 3, 4), 4)[1]
    n = int(places.max())
    for size in (96, 95):
        z, w, r, g = normal(1, n, size), normal(2, 50, 3), normal(3, 50, size), normal(4, 50, size)
        y, mass, gz, gw, wmass = exact_combine(z, w, places, r, g)

        def apart(a, by=5, off=2):
            wide = gt.GPUTensor(a.shape[0], a.shape[1] + by).fill(np.nan)
            v = wide.narrow(2, 1 + off, a.shape[1])
            v.copy(gt.gpu(a))
            return v

        def turned(a):
            return gt.gpu(np.ascontiguousarray(a.T)).t()
        for lay in (apart, turned):
            m = gt.nn.Combine()
            input = [lay(z), lay(w), lay(f32(places)), lay(r)]
            assert np.all(np.abs(m.forward(input).float() - y) <= 4 * U * mass)
            back = m.backward(input, lay(g))
            assert np.all(np.abs(back[0].float() - gz) <= U * np.abs(gz)) and np.all(np.abs(back[1].float() - gw) <= 16 * U * wmass)


# ------------------------------------------------------------------ more values than 32 bits count
def test_rows_beyond_32_bits(gt):
    """525000 rows of 4096 values, turned round: the last token goes to the first expert."""
    tokens, size, groups = 525000, 4096, 4
    x = torch.zeros(tokens, size, device="cuda")
    x[:, 0] = torch.arange(tokens, device="cuda")
    x[-3:] = torch.randn(3, size, device="cuda")
    e = np.repeat([4, 3, 2, 1], tokens // 4).reshape(-1, 1)
    order, places, counts = plan(e, groups)
    torch.cuda.synchronize()
    L = gt.lib()
    st = L.THGPUStorage_newWithData(x.data_ptr(), x.numel())
    X = gt.GPUTensor(_ptr=L.THGPUTensor_newWithStorage1d(st, 0, x.numel(), 1)).view(tokens, size)
    L.THGPUStorage_free(st)
    m = gt.nn.Dispatch(groups)
    E = gt.gpu(f32(e))
    rows, told = m.forward([X, E])
    assert np.array_equal(told, counts) and np.array_equal(m.positions.float(), places)
    assert np.array_equal(rows.select(2, 1).float()[:-tokens // 4], x[:, 0].cpu().numpy()[order][:-tokens // 4])
    at = int(places[-1, 0])
    assert np.array_equal(rows.narrow(1, at - 2, 3).float(), x[-3:].cpu().numpy())
    gx = m.backward([X, E], [rows, None])[0]
    assert np.array_equal(gx.narrow(1, tokens - 2, 3).float(), x[-3:].cpu().numpy()) and np.array_equal(gx.select(2, 1).float(), x[:, 0].cpu().numpy())
    del x, X, gx
    m.gradRows = gt.GPUTensor()
    torch.cuda.empty_cache()
    c = gt.nn.Combine()
    w = gt.GPUTensor(tokens, 1).fill(2.0)
    y = c.forward([rows, w, m.positions])
    assert np.array_equal(y.narrow(1, tokens - 2, 3).float(), 2 * rows.narrow(1, at - 2, 3).float())
    assert np.array_equal(y.select(2, 1).float()[places[:, 0] - 1 >= 0], 2 * rows.select(2, 1).float()[places[:, 0] - 1])
    back = c.backward([rows, w, m.positions], y)
    assert np.array_equal(back[0].narrow(1, at - 2, 3).float(), 4 * rows.narrow(1, at - 2, 3).float())
    dot = (rows.narrow(1, at - 2, 3).float().astype(np.float64) ** 2).sum(1) * 2
    assert np.all(np.abs(back[1].float()[-3:, 0] - dot) <= (4096 / 32 + 10) * U * dot)
