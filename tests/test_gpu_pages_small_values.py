"""Caches of 8-bit pages whose values are small, or of very different sizes along a sequence: outputs as close to 64 bits as
those of ordinary values."""
import numpy as np
import pytest

from tests.pages_model import Model

pytestmark = pytest.mark.gpu

# Errors of scores and sums are those of the step's other tests, 2e-5 of the largest output at the worst.  A weight times
# its row's scale is held to half of 2^-126, or 2^-31 of the largest of 64 positions: with values' rows of 2^-88 at least
# (3e-27), scales of 2^-95 and weights of 2^-4 at their largest, to 2^-28 of that, which over the 6000 rows below and if all
# fell the same way is 2.3e-5 of the largest value, and near 3e-7 as they come.
TOL = 2e-5


@pytest.fixture(scope="module", autouse=True)
def _needs_gpu(hip_device):
    return hip_device


def _check(m, lens, sizes, new):
    """A step with values whose rows have the given sizes, [len] of each sequence, and the new ones'."""
    m.fill(lens)
    for i, n in enumerate(lens):
        k, v = (m.rng.standard_normal((n, m.nkv * m.hd)).astype(np.float32) for _ in range(2))
        m.write(i, 0, 0, k, v * np.asarray(sizes[i], np.float32)[:, None])
    m.reserve(lens, [n + 1 for n in lens])
    q, k, v = m.tokens(len(lens))
    v *= np.asarray(new, np.float32)[:, None]
    got, want = m.h.step(0, lens, q, k, v), m.want(0, lens, q, k, v)
    for i in range(len(lens)):
        assert np.isfinite(got[i]).all()
        e = np.abs(got[i] - want[i]).max() / np.abs(want[i]).max()
        assert e <= TOL, (i, e)


@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 128), (16, 1, 64), (3, 1, 64)])
@pytest.mark.parametrize("n", [0, 40, 400, 6000])
@pytest.mark.parametrize("scale", [1e-21, 1e-23, 1e-25, 3e-27])
def test_small_values(scale, n, nh, nkv, hd):
    m = Model(nh, nkv, hd, 6100, 1, "q8", 32, key=n)
    with m.h:
        _check(m, [n], [[scale] * n], [scale])


@pytest.mark.parametrize("first,last", [(1e-26, 1e26), (1e26, 1e-26), (1e-26, 1e36), (1e36, 1e-26), (1.0, 1e-26), (1e-20, 1e-26)])
@pytest.mark.parametrize("n", [100, 700, 6000])
def test_values_of_many_sizes(first, last, n):
    """Sizes that rise or fall along a sequence, and that jump from row to row."""
    m = Model(8, 2, 128, 6100, 3, "q8", 32, key=n)
    with m.h:
        ramp = np.exp(np.linspace(np.log(first), np.log(last), n))
        jumps = np.where(m.rng.random(n) < 0.1, first, last)
        late = np.where(np.arange(n) < n - 70, first, last)
        _check(m, [n, n, n], [ramp, jumps, late], [last, first, 1.0])


def test_small_values_in_an_unequal_batch():
    """Enough rows for a launch that shares the tiles out over the chip."""
    m = Model(32, 8, 128, 4100, 24, "q8", 16)
    with m.h:
        lens = m.rng.integers(300, 4000, 24).tolist()
        lens[3] = 0
        sizes = [10.0 ** m.rng.integers(-25, 30) for _ in lens]
        _check(m, lens, [[s] * n for s, n in zip(sizes, lens)], sizes)


@pytest.mark.parametrize("low,high", [(1e36, 1e-26), (1e-26, 1e36), (1e36, 1.0), (1.0, 1e-26)])
@pytest.mark.parametrize("n", [60, 500, 6000])
@pytest.mark.parametrize("order", ["low first", "high first", "one high"])
def test_sizes_behind_the_scores(order, n, low, high):
    """Rows of one size with scores far below those of the rows of another, which alone count: in every order, so that the
    reference moves before or after the values change."""
    m = Model(4, 1, 128, 6100, 1, "q8", 16, key=n)
    with m.h:
        m.fill([n])
        k, v = (m.rng.standard_normal((n, 128)).astype(np.float32) for _ in range(2))
        q, kn, vn = m.tokens(1)
        at = np.arange(n)
        counts = {"low first": at >= n // 2, "high first": at < n // 2, "one high": at == n // 3}[order]
        y = m.turned(q[0], n).reshape(4, 128).mean(axis=0)
        y *= 3000.0 / (y @ y) * np.sqrt(128)  # (a score of about 3000 of the heads' mean)
        k = np.where(counts[:, None], k * 0.1, k * 0.1 - y.astype(np.float32))
        # every head has the same query, so that all scores part
        q[:] = np.tile(q[0].reshape(4, 128).mean(axis=0), 4)
        kn[:], vn[:] = 0, 0
        v = v * np.where(counts, high, low).astype(np.float32)[:, None]
        m.write(0, 0, 0, k, v)
        m.reserve([n], [n + 1])
        got, want = m.h.step(0, [n], q, kn, vn), m.want(0, [n], q, kn, vn)
        assert np.isfinite(got).all()
        e = np.abs(got - want).max() / np.abs(want).max()
        assert e <= TOL, e
