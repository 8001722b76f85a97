"""nn.Router against its definition in 64 bits, its gradient against the formula's and against differences."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def gt():
    import mcw_cppamp_torch_b200 as gt
    return gt


def choose(x, k):
    """Places of each row's k largest, from 1, 0 where there is no open one left: a NaN first, equal ones by their place."""
    key = np.where(np.isnan(x), np.inf, x.astype(np.float64))
    nan_first = np.where(np.isnan(x), 0, 1)
    order = np.stack([np.lexsort((np.arange(x.shape[1]), -key[r], nan_first[r])) for r in range(len(x))])[:, :k] if len(x) else np.zeros((0, k), np.int64)
    open_ = np.take_along_axis(~np.isneginf(x), order, 1)
    return np.where(open_, order + 1, 0)


def soft(x, ids, normalize):
    """The whole softmax that the weights are of, in 64 bits: over the chosen scores or over all."""
    x = x.astype(np.float64)
    if normalize:
        on = np.zeros(x.shape, bool)
        for r in range(len(x)):
            on[r, ids[r][ids[r] > 0] - 1] = True
        x = np.where(on, x, -np.inf)
    with np.errstate(invalid="ignore"):
        top = x.max(1, keepdims=True)
        e = np.where(np.isneginf(x), 0.0, np.exp(x - np.where(np.isneginf(top), 0.0, top)))
        total = e.sum(1, keepdims=True)
        return e / np.where(total == 0, 1.0, total)


def spread_of(x):
    """How far a row's scores are apart: the difference that the exponential is taken of carries half a step of it."""
    f = np.where(np.isfinite(x), x, np.nan)
    return np.nan_to_num(np.nanmax(f, 1, initial=-1e30, where=~np.isnan(f)) - np.nanmin(f, 1, initial=1e30, where=~np.isnan(f)), neginf=0.0).clip(0)[:, None]


def scores(seed, rows, experts, closed=0.0, empty=0):
    r = np.random.RandomState(seed)
    x = (2 * r.standard_normal((rows, experts))).astype(np.float32)
    x[r.random_sample(x.shape) < closed] = -np.inf
    x[rows - empty:] = -np.inf
    return x


def check(gt, x, k, normalize, g=None, lay=lambda t: t):
    m = gt.nn.Router(k, normalize)
    w, e = m.forward(lay(gt.gpu(x)))
    ids = choose(x, k)
    assert np.array_equal(e.float(), ids.astype(np.float32))
    p = soft(x, ids, normalize)
    want = np.where(ids > 0, np.take_along_axis(p, np.maximum(ids - 1, 0), 1), 0.0)
    # each exponential: half a step of the difference, two of its own; two sums' worth of them in the quotient, the sum's own steps (V a lane and 5), the quotient's
    rel = (2 * (spread_of(x) + 4) + x.shape[1] / 32 + 8) * U
    assert np.all(np.abs(w.float() - want) <= rel * want + 1e-37)
    if g is None:
        return m
    gi = m.backward(lay(gt.gpu(x)), [lay(gt.gpu(g)), None]).float()
    G = np.zeros(x.shape)
    for i in range(k):
        r = np.nonzero(ids[:, i])[0]
        G[r, ids[r, i] - 1] += g[r, i]
    dot, mass = (p * G).sum(1, keepdims=True), (p * np.abs(G)).sum(1, keepdims=True)
    assert np.all(np.abs(gi - p * (G - dot)) <= p * (np.abs(G) + mass) * (3 * rel + 48 * U) + 1e-37)
    return m


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("rows,experts,k", [(1, 1, 1), (1, 64, 8), (7, 33, 6), (9, 32, 32), (300, 77, 5), (260, 128, 2), (65, 256, 8), (17, 516, 9), (3, 1024, 32), (5, 1023, 31),
                                            (2000, 16, 2), (11, 2, 1), (8, 4, 4)])
def test_against_the_definition(gt, rows, experts, k, normalize):
    x = scores(rows + experts, rows, experts)
    check(gt, x, k, normalize, np.random.RandomState(3).standard_normal((rows, k)).astype(np.float32))


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("experts,k", [(8, 4), (77, 6), (300, 32), (128, 3)])
def test_closed_experts(gt, experts, k, normalize):
    """Rows with fewer open experts than they are to have, and with none; gradients of empty slots are not looked at."""
    x = scores(5, 120, experts, 0.5, 9)
    x[3, 1:] = -np.inf
    x[4] = -np.inf
    x[5, :experts - 2] = -np.inf
    g = np.random.RandomState(3).standard_normal((120, k)).astype(np.float32)
    ids = choose(x, k)
    assert (ids == 0).any() and (ids == 0).all(1).sum() >= 10
    g[ids == 0] = np.nan
    clean = np.where(ids == 0, 0, g).astype(np.float32)
    m = check(gt, x, k, normalize, clean)
    a = m.gradInput.float()
    assert np.array_equal(a, m.backward(gt.gpu(x), gt.gpu(g)).float()) and not a[np.isneginf(x)].any()


@pytest.mark.parametrize("experts,k", [(64, 8), (130, 32), (9, 9), (130, 8), (96, 16), (97, 17), (256, 8), (300, 16), (512, 1), (1000, 6), (1024, 16)])
@pytest.mark.parametrize("levels", [3, 40, 1000])
def test_equal_scores(gt, experts, k, levels):
    """By their place, zeros of both signs alike: many of each score, so that more than 32 may be as large as the last chosen one, and few."""
    x = np.random.RandomState(0).randint(-levels, levels, (200, experts)).astype(np.float32)
    x[::2][x[::2] == 0] = -0.0
    x[5], x[6], x[7, ::2] = 1.0, 0.0, -0.0
    x[7, 1::2] = 0.0
    x[8], x[8, experts // 2] = -np.inf, 0.0
    check(gt, x, k, True)
    check(gt, x, k, False)


@pytest.mark.parametrize("experts", [16, 33, 64, 77, 128, 200, 256])
@pytest.mark.parametrize("normalize", [True, False])
def test_many_rows(gt, experts, normalize):
    """So many rows that several share a warp: the same choices as of a few, weights but for the order of their sums."""
    r = np.random.RandomState(experts)
    parts = [scores(experts, 200, experts), scores(1, 61, experts, 0.6, 3), r.randint(-2, 3, (50, experts)).astype(np.float32),
             r.randint(-60, 60, (80, experts)).astype(np.float32), scores(2, 20, experts)]
    parts[4][3, 5], parts[4][7, [3, 9]], parts[4][11, 2], parts[4][15, 2:] = np.nan, (np.nan, np.inf), np.inf, -np.inf
    parts[2][::2][parts[2][::2] == 0] = -0.0
    x = np.concatenate(parts)
    times = 24000 // len(x) + 1
    X = np.concatenate([np.tile(x, (times, 1)), x[:3]])
    for k in (1, 2, 6, 8):
        w, e = (t.float() for t in gt.nn.Router(k, normalize).forward(gt.gpu(x)))
        assert np.array_equal(e, choose(x, k))
        W, E = (t.float() for t in gt.nn.Router(k, normalize).forward(gt.gpu(X)))
        assert np.array_equal(E, np.concatenate([np.tile(e, (times, 1)), e[:3]]))
        want = np.concatenate([np.tile(w, (times, 1)), w[:3]])
        # the sums of up to 256 exponentials in two orders, 8 + 5 and 32 + 3 additions deep, and the quotients' own half step each
        assert np.array_equal(np.isnan(W), np.isnan(want)) and np.all(np.abs(W - want)[~np.isnan(W)] <= (50 * U * np.abs(want))[~np.isnan(W)])
    flat = gt.GPUTensor(X.size + 1)
    off = flat.narrow(1, 2, X.size).view(*X.shape)             # no 16-byte addresses
    off.copy(X)
    assert np.array_equal(gt.nn.Router(8, normalize).forward(off)[1].float(), E)


def test_scores_that_are_not_finite(gt):
    x = scores(1, 6, 40)
    x[0, 7] = np.nan
    x[1, [3, 9]] = np.nan, np.inf
    x[2, 5] = np.inf
    x[3, :] = -np.inf
    x[3, 8] = np.nan
    x[4, ::3] = -np.inf
    for normalize in (True, False):
        m = gt.nn.Router(4, normalize)
        w, e = (t.float() for t in m.forward(gt.gpu(x)))
        assert np.array_equal(e, choose(x, 4))
        assert np.isnan(w[[0, 1]]).all() and np.isnan(w[2, 0]) and np.isnan(w[3, 0])
        assert not w[3, 1:].any() and np.isfinite(w[4:]).all()
        gi = m.backward(gt.gpu(x), gt.gpu(np.ones((6, 4), np.float32))).float()
        assert np.isfinite(gi[4:]).all() and not gi[4, ::3].any()
    big = np.float32(3e38)
    x = np.array([[big, -big, 0, big], [-big, -big, -big, -np.inf], [1e-45, 0, -1e-45, -np.inf]], np.float32)
    for normalize in (True, False):
        w, e = (t.float() for t in gt.nn.Router(3, normalize).forward(gt.gpu(x)))
        assert np.array_equal(e, [[1, 4, 3], [1, 2, 3], [1, 2, 3]])
        assert np.allclose(w, [[.5, .5, 0], [1 / 3] * 3, [1 / 3] * 3], rtol=1e-6, atol=0)


@pytest.mark.parametrize("normalize", [True, False])
def test_strides(gt, normalize):
    """Rows apart, rows at addresses that are no multiple of 16 bytes, and a transposed matrix."""
    x = scores(2, 50, 64)
    g = np.random.RandomState(3).standard_normal((50, 4)).astype(np.float32)

    def apart(by, off):
        def lay(t):
            wide = gt.GPUTensor(t.size(1), t.size(2) + by).fill(np.nan)
            v = wide.narrow(2, 1 + off, t.size(2))
            v.copy(t)
            return v
        return lay
    plain = check(gt, x, 4, normalize, g)
    for lay in (apart(4, 0), apart(8, 4), apart(3, 1), lambda t: gt.gpu(np.ascontiguousarray(t.float().T)).t()):
        m = check(gt, x, 4, normalize, g, lay)
        for a, b in zip(m.output + [m.gradInput], plain.output + [plain.gradInput]):
            assert np.allclose(a.float(), b.float(), rtol=1e-5, atol=1e-7)
    m = gt.nn.Router(4, normalize)
    room = gt.GPUTensor(50 * 64 + 1)
    m.gradInput = room.narrow(1, 2, 50 * 64).view(50, 64)
    m.forward(gt.gpu(x))
    assert np.allclose(m.backward(gt.gpu(x), gt.gpu(g)).float(), plain.gradInput.float(), rtol=1e-5, atol=1e-7)


@pytest.mark.parametrize("normalize", [True, False])
def test_differences(gt, normalize):
    """Of sum(g w) along a direction that leaves the order of the scores as it is."""
    r = np.random.RandomState(7)
    x = np.stack([r.permutation(24) for _ in range(5)]).astype(np.float32) * 0.25
    g, d = r.standard_normal((5, 6)).astype(np.float32), r.uniform(-1, 1, x.shape).astype(np.float32)
    h = 2.0 ** -5
    m = gt.nn.Router(6, normalize)

    def loss(v):
        w, e = m.forward(gt.gpu(v.astype(np.float32)))
        return (w.float().astype(np.float64) * g).sum()
    numeric = (loss(x + h * d) - loss(x - h * d)) / (2 * h)
    m.forward(gt.gpu(x))
    gi = m.backward(gt.gpu(x), gt.gpu(g)).float().astype(np.float64)
    # rounding: 40 half steps of each weight over 2 h; the third derivative of a softmax along a direction of size 1 is below 8 of its row's largest |g|
    assert abs(numeric - (gi * d).sum()) <= 40 * U * np.abs(g).sum() / (2 * h) + 8 * np.abs(g).max(1).sum() * h * h / 6


def test_no_rows_and_results_that_change_size(gt):
    m = gt.nn.Router(3)
    w, e = m.forward(gt.GPUTensor())
    assert w.nElement() == e.nElement() == 0
    assert m.backward(gt.GPUTensor(), gt.GPUTensor()).nElement() == 0
    for rows in (9, 2, 30):
        x = scores(rows, rows, 20)
        w, e = m.forward(gt.gpu(x))
        assert w.size() == (rows, 3) and np.array_equal(e.float(), choose(x, 3))
        assert m.backward(gt.gpu(x), gt.gpu(np.ones((rows, 3), np.float32))).size() == (rows, 20)


@pytest.mark.parametrize("experts", [256, 300])
def test_more_values_than_32_bits_count(gt, experts):
    """Rows at both ends of more than 2^31 scores, as by themselves, with equal scores between them."""
    rows, k = 2 ** 31 // experts + 1009, 2
    few = scores(4, 40, experts)
    x = gt.GPUTensor(rows, experts).fill(0.5)
    x.narrow(1, 1, 20).copy(few[:20])
    x.narrow(1, rows - 19, 20).copy(few[20:])
    gw = gt.GPUTensor(rows, k).fill(0.0)
    g = np.random.RandomState(1).standard_normal((40, k)).astype(np.float32)
    gw.narrow(1, 1, 20).copy(g[:20])
    gw.narrow(1, rows - 19, 20).copy(g[20:])
    m, small = gt.nn.Router(k, False), gt.nn.Router(k, False)
    got, want = m.forward(x), [t.float() for t in small.forward(gt.gpu(few))]

    def ends(t):
        return np.concatenate([t.narrow(1, 1, 20).float(), t.narrow(1, rows - 19, 20).float()])
    assert np.array_equal(ends(got[1]), want[1]) and np.all(np.abs(ends(got[0]) - want[0]) <= 50 * U * want[0])
    between = got[1].narrow(1, rows // 2, 3).float()
    assert np.array_equal(between, np.tile([1, 2], (3, 1)))
    gi, wg = ends(m.backward(x, gw)), small.backward(gt.gpu(few), gt.gpu(g)).float()
    # two evaluations of p (g - sum g w), whose p and w are those above
    p = soft(few, choose(few, k), False)
    assert np.all(np.abs(gi - wg) <= 2 * 60 * U * p * (np.abs(g).max(1) * 2)[:, None] + 1e-37)
