"""Caches of pages through the C ABI: the step over them, the tables' calls and the choice of pages, against a plain
model whose attention is in 64 bits."""
import errno

import numpy as np
import pytest

from leap_amd.attention import LeapError, PagedAttention
from tests.helpers import attention_f64, rng_for, rope_f32
from tests.pages_model import Model

pytestmark = pytest.mark.gpu

# Outputs are weighted means of values: with |v| <= V their error is at most
# 2 V (largest error of a score) + V (terms of the sums).  A score of these
# inputs is a sum of up to 128 products with sum |q_i k_i| / sqrt(hd) near 15
# (q has twice the spread of k), in two chains of 64 additions at most:
# under 15 * 40 * 2^-24 < 4e-5 if all of 40 roundings fell the same way, and
# near 1e-6 as they come; exp, weights and sums add a few 2^-24.  (8 bits: q
# to 2^-30 of its largest, exact products, a few roundings.)  2e-5 of the
# largest output is asserted.
TOL = 2e-5


@pytest.fixture(scope="module", autouse=True)
def _needs_gpu(hip_device):
    return hip_device


def _ptr(t):
    return t.data_ptr()


def _dev(*arrays):
    import torch
    return [torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in arrays]


def _i32(x):
    import torch
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def _close(got, want, tol=TOL):
    assert np.isfinite(got).all()
    e = np.abs(got - want).max() / np.abs(want).max()
    assert e <= tol, e


def _refused(fragment, fn, *args, code=errno.EINVAL):
    with pytest.raises(LeapError) as e:
        fn(*args)
    assert e.value.code == -code and fragment in str(e.value), str(e.value)


SHAPES = [(32, 8, 128), (32, 4, 64), (4, 4, 128), (3, 1, 64), (6, 3, 128), (32, 2, 128), (16, 2, 64), (16, 1, 64)]


@pytest.mark.parametrize("cache", ["f32", "q8"])
@pytest.mark.parametrize("nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("pos,page_rows", [
    ([0], 16), ([15], 16), ([16], 16), ([200], 32), ([63], 64), ([64], 128), ([300], 16), ([777], 64),
    ([0, 1, 64, 1000, 1499], 16), ([127, 128, 129, 31, 17, 0, 255], 32),
])
def test_step_matches_64_bits(nh, nkv, hd, pos, page_rows, cache):
    m = Model(nh, nkv, hd, 1500, len(pos), cache, page_rows, layers=2, key=sum(pos))
    with m.h:
        m.fill(pos)
        m.reserve(pos, [p + 1 for p in pos])
        for layer in (1, 0):
            q, k, v = m.tokens(len(pos))
            _close(m.h.step(layer, pos, q, k, v), m.want(layer, pos, q, k, v))
        m.check_rows([p + 1 for p in pos])
        m.check_state()


@pytest.mark.parametrize("cache", ["f32", "q8"])
@pytest.mark.parametrize("nh,nkv,hd,n_seq,pos", [
    (32, 8, 128, 1, 5000), (32, 8, 128, 1, 12345), (8, 1, 128, 1, 20000), (8, 1, 64, 1, 33000), (32, 4, 64, 3, 4100), (64, 8, 128, 9, 2500),
    (16, 1, 128, 2, 9000),
])
def test_step_over_long_caches(nh, nkv, hd, n_seq, pos, cache):
    """Many runs a group, and groups spread over the XCDs."""
    m = Model(nh, nkv, hd, pos + 1, n_seq, cache, 64, spare=0)
    with m.h:
        at = [pos - 97 * i for i in range(n_seq)]
        m.fill(at)
        m.reserve(at, [p + 1 for p in at])
        q, k, v = m.tokens(n_seq)
        _close(m.h.step(0, at, q, k, v), m.want(0, at, q, k, v))


@pytest.mark.parametrize("cache", ["f32", "q8"])
def test_many_short_sequences(cache):
    n = 300
    m = Model(8, 2, 64, 96, n, cache, 16)
    with m.h:
        pos = m.rng.integers(0, 96, n).tolist()
        m.fill(pos)
        m.reserve(pos, [p + 1 for p in pos])
        q, k, v = m.tokens(n)
        _close(m.h.step(0, pos, q, k, v), m.want(0, pos, q, k, v))
        m.check_rows([p + 1 for p in pos])


@pytest.mark.parametrize("cache", ["f32", "q8"])
@pytest.mark.parametrize("bounds", [False, True])
@pytest.mark.parametrize("seed", range(4))
def test_tables_and_contents_follow_the_model(seed, bounds, cache):
    """Reservations, forks, cuts and compactions in any order: tables, references and every row after each."""
    rng = rng_for(0x7461626C, seed)
    page_rows, n_seq = (16, 32)[seed % 2], 7
    m = Model(6, 3, 64, 200, n_seq, cache, page_rows, layers=2, bounds=bounds, key=seed, n_pages=(45, 37)[seed % 2])
    lens = [0] * n_seq
    with m.h:
        for op in range(70):
            what = rng.choice(["grow", "grow", "grow", "fork", "cut", "compact", "rewrite"])
            if what in ("grow", "rewrite"):
                n = int(rng.integers(1, n_seq + 1))
                begin = [x if what == "grow" else int(rng.integers(0, x + 1)) for x in lens[:n]]
                end = [min(200, x + int(rng.choice([0, 0, 1, 5, 40]))) for x in begin]
                if not m.p.reserve(begin, end):
                    _refused("too few", m.h.reserve, begin, end, code=errno.ENOMEM)
                    m.check_state()
                    continue
                m.h.reserve(begin, end)
                for i in range(n):
                    if end[i] > begin[i]:
                        for l in range(2):
                            k, v = (rng.standard_normal((end[i] - begin[i], 192)).astype(np.float32) for _ in range(2))
                            m.write(i, l, begin[i], k, v)
                    lens[i] = max(lens[i], end[i]) if end[i] > begin[i] else lens[i]
            elif what == "compact":
                assert m.h.compact() == m.p.compact()
            else:
                n = int(rng.integers(1, n_seq + 1))
                parent = None if what == "cut" else rng.integers(0, n_seq, n).tolist()
                rows = [int(rng.integers(0, lens[i if parent is None else parent[i]] + 1)) if rng.random() < 0.4
                        else lens[i if parent is None else parent[i]] for i in range(n)]
                m.fork(parent, rows)
                lens[:n] = rows
            m.check_state()
            m.check_rows(lens)
        m.h.clear()
        table, refs = m.h.state()
        assert (table == -1).all() and not refs.any()


def test_the_last_of_all_who_share_a_page_keeps_it():
    m = Model(8, 2, 64, 64, 4, page_rows=16)
    with m.h:
        m.fill([20, 0, 0, 0])
        m.fork([0, 0, 0, 0], [20] * 4)
        m.check_state()
        m.reserve([20] * 4, [21] * 4)
        m.check_state()
        table, refs = m.h.state()
        assert refs[table[0, 0]] == 4 and len(set(table[:, 1])) == 4
        m.check_rows([20] * 4)
        # and where only some of them ask, all of these copy
        m.fork([0, 0, 0, 0], [20] * 4)
        m.reserve([20, 20], [21, 21])
        m.check_state()
        m.check_rows([20] * 4)


def test_a_pool_that_is_too_small_changes_nothing():
    import torch
    m = Model(8, 2, 64, 128, 3, page_rows=16, n_pages=5)
    with m.h:
        m.fill([32, 16, 0])
        m.fork([0, 1, 0], [32, 16, 32])  # the third shares both pages of the first
        m.check_state()
        begin, end = _i32([30, 16, 16]), _i32([33, 17, 17])  # 2 + 1 pages, and one more: the pool has 2
        status = _i32([7, 7, 7])
        m.h.reserve_async(3, _ptr(begin), _ptr(end), _ptr(status), torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert status.tolist() == [-errno.ENOMEM] * 3
        m.check_state()
        _refused("too few", m.h.reserve, [30, 16, 16], [33, 17, 17], code=errno.ENOMEM)
        m.check_state()
        m.check_rows([32, 16, 32])
        m.reserve([30], [32])  # (what fits still does)
        m.check_state()
        m.check_rows([32, 16, 32])


def test_bad_ranges_and_parents_on_the_device_are_left_out():
    import torch
    m = Model(8, 2, 64, 100, 6, page_rows=32)
    with m.h:
        m.fill([40, 33, 0, 10, 0, 0])
        begin, end = _i32([-1, 33, 5, 0, 90, 7]), _i32([4, 70, 4, 101, 100, 7])
        status = _i32([7] * 6)
        s = torch.cuda.current_stream().cuda_stream
        m.h.reserve_async(6, _ptr(begin), _ptr(end), _ptr(status), s)
        torch.cuda.synchronize()
        bad = -errno.EINVAL
        assert status.tolist() == [bad, 0, bad, bad, 0, 0]
        assert m.p.reserve([0, 33, 0, 0, 90, 0], [0, 70, 0, 0, 100, 0])
        m.check_state()
        m.h.reserve_async(6, _ptr(begin), _ptr(end), 0, s)
        m.check_state()
        parent, rows = _i32([-1, 6, 1, 0, 0, 1 << 30]), _i32([0, 0, 40, -1, 101, 3])
        m.h.fork_async(6, _ptr(parent), _ptr(rows), s)
        torch.cuda.synchronize()
        m.p.fork([0, 1, 1, 3, 4, 5], [100, 100, 40, 100, 100, 100])
        m.check_state()


@pytest.mark.parametrize("cache", ["f32", "q8"])
def test_a_step_needs_pages_of_its_own(cache):
    """A shared page, a missing one, one missing before: NaN, and nothing is written; the others are served."""
    import torch
    m = Model(8, 2, 128, 128, 6, cache, 16)
    with m.h:
        m.fill([20, 30, 40, 17, 33, 9])
        m.fork([0, 0, 2, 3, 4, 5], [20, 20, 40, 16, 33, 9])     # 0 and 1 share; 3 has no page for row 16
        m.reserve([0, 0, 48, 0, 0, 0], [0, 0, 49, 0, 0, 0])     # (2: rows 40..47 are there, 48 too)
        m.fork(None, [20, 20, 49, 16, 16, 9])                   # 4: pages from row 16 on are gone
        m.reserve([0, 0, 0, 0, 33, 0], [0, 0, 0, 0, 34, 0])     # but for the page of row 33
        pos = [19, 12, 48, 16, 33, 8]
        q, k, v = m.tokens(6)
        before = [m.h.read(i, 0, 0, n) for i, n in ((0, 20), (1, 20))]
        got = m.h.step(0, pos, q, k, v)
        assert np.isnan(got[[0, 1, 3, 4]]).all()
        for i, (kk, vv) in enumerate(before):
            assert np.array_equal(m.h.read(i, 0, 0, 20)[0], kk) and np.array_equal(m.h.read(i, 0, 0, 20)[1], vv)
        assert np.isfinite(got[[2, 5]]).all()
        assert np.isnan(m.h.read(3, 0, 16, 17)[0]).all() and np.isnan(m.h.read(4, 0, 16, 32)[1]).all()
        # positions on the device that are out of range
        m2 = Model(8, 2, 128, 128, 4, cache, 16, key=1)
        with m2.h:
            m2.fill([50] * 4)
            m2.reserve([50] * 4, [51] * 4)
            q, k, v = m2.tokens(4)
            d, out = _dev(q, k, v), torch.full((5, 8 * 128), 3.0, device="cuda")
            at = _i32([50, -1, 128, 61])
            m2.h.step_async(0, 4, _ptr(at), 60, *map(_ptr, d), _ptr(out), torch.cuda.current_stream().cuda_stream)
            torch.cuda.synchronize()
            got = out.cpu().numpy()
            assert np.isnan(got[1:4]).all() and (got[4] == 3.0).all()
            _close(got[:1], m2.want(0, [50], q, k, v))
            m2.check_rows([51, 50, 50, 50])


@pytest.mark.parametrize("cache", ["f32", "q8"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, 1e38])
def test_what_recycled_pages_held_does_not_matter(cache, bad):
    """Rows behind a sequence's last, in its last page, of an earlier tenant."""
    m = Model(16, 4, 128, 256, 2, cache, 64, bounds=True)
    with m.h:
        m.reserve([0, 0], [256, 200])
        rows = np.full((256, 512), bad, np.float32)
        m.h.write(0, 0, 0, rows, rows)
        m.h.write(1, 0, 0, rows[:200], rows[:200])
        m.fork(None, [0, 0])
        for pos in ([0, 0], [5, 70], [63, 64], [130, 17]):
            m.fork(None, [0, 0])
            m.fill(pos)
            m.reserve(pos, [p + 1 for p in pos])
            q, k, v = m.tokens(2)
            _close(m.h.step(0, pos, q, k, v), m.want(0, pos, q, k, v))
            q, k, v = m.tokens(2)
            got, picked = m.h.step_sparse(0, pos, 2, q, k, v)
            want, pages = m.want_sparse(0, pos, 2, q, k, v)
            assert np.array_equal(picked, pages)
            _close(got, want)


@pytest.mark.parametrize("cache", ["f32", "q8"])
@pytest.mark.parametrize("where,bad", [("k", np.inf), ("k", np.nan), ("v", -np.inf), ("v", np.nan), ("new k", np.nan), ("new v", np.inf),
                                       ("q", np.nan), ("q", np.inf)])
def test_rows_that_are_not_finite(where, bad, cache):
    """NaN for the KV head that sees them, and for no other."""
    nh, nkv, hd = 16, 4, 128
    m = Model(nh, nkv, hd, 512, 2, cache, 16)
    with m.h:
        pos = [300, 40]
        m.fill(pos)
        m.reserve(pos, [p + 1 for p in pos])
        q, k, v = m.tokens(2)
        clean = m.want(0, pos, q, k, v).reshape(2, nkv, -1)
        at = 2 * hd + 7
        if where in ("k", "v"):
            for x in ((m.h.write(0, 0, 123, *[r if w == where else None for w, r in (("k", _bad_row(m, 0, bad, at)), ("v", _bad_row(m, 1, bad, at)))]),)):
                assert x is None
        else:
            {"new k": k, "new v": v, "q": q}[where][0, (2 * 4 * hd + 7) if where == "q" else at] = bad
        got = m.h.step(0, pos, q, k, v).reshape(2, nkv, -1)
        if where == "q":
            assert np.isnan(got[0, 2, :hd]).all()
            got[0, 2, :hd] = clean[0, 2, :hd]
        elif cache == "f32" and where in ("v", "new v"):
            # (one element of V: that dim of the heads)
            assert not np.isfinite(got[0, 2].reshape(-1, hd)[:, 7]).any()
            got[0, 2].reshape(-1, hd)[:, 7] = clean[0, 2].reshape(-1, hd)[:, 7]
        elif where == "k" and cache == "f32" and np.isinf(bad):
            # (a score of +-inf by q's sign: the row alone has NaN or none of the weight)
            x = got[0, 2].reshape(-1, hd)
            assert np.isnan(x).all(axis=1).any() or np.isfinite(x).all()
            got[0, 2] = clean[0, 2]
        else:
            assert np.isnan(got[0, 2]).all()
            got[0, 2] = clean[0, 2]
        _close(got, clean)


def _bad_row(m, which, bad, at):
    row = m.p.row(0, 0, 123)[which].astype(np.float32).copy()
    row[at] = bad
    return row[None]


@pytest.mark.parametrize("cache", ["f32", "q8"])
@pytest.mark.parametrize("scale", [1e-20, 1e-10, 1e10, 1e30])
def test_values_of_any_size(scale, cache):
    m = Model(8, 2, 128, 512, 1, cache, 32, key=int(np.log10(scale)) + 50)
    with m.h:
        m.fill([400])
        k, v = (m.rng.standard_normal((400, 256)).astype(np.float32) for _ in range(2))
        m.write(0, 0, 0, k, v * np.float32(scale))
        m.reserve([400], [401])
        q, k, v = m.tokens(1)
        v *= np.float32(scale)
        _close(m.h.step(0, [400], q, k, v), m.want(0, [400], q, k, v))


@pytest.mark.parametrize("cache", ["f32", "q8"])
def test_the_largest_floats_average(cache):
    """A mean of values at fp32's end is finite."""
    m = Model(8, 2, 64, 2048, 1, cache, 16)
    with m.h:
        m.fill([2000])
        top = np.float32(3.3e38)
        m.write(0, 0, 0, np.zeros((2000, 128), np.float32), np.full((2000, 128), top))
        m.reserve([2000], [2001])
        q, k, _ = m.tokens(1)
        k *= 0
        v = np.full((1, 128), top)
        got = m.h.step(0, [2000], q, k, v)
        # (8 bits: 127 * (top / 127) rounds once more)
        assert np.abs(got / top - 1).max() < 1e-6


@pytest.mark.parametrize("cache", ["f32", "q8"])
@pytest.mark.parametrize("nh,nkv,hd", [(32, 8, 128), (8, 2, 64), (16, 1, 128)])
def test_scores_far_apart(nh, nkv, hd, cache):
    """Keys a thousand times the others, at places that move the reference again and again."""
    m = Model(nh, nkv, hd, 3000, 1, cache, 16)
    with m.h:
        m.fill([2900])
        k, v = (m.rng.standard_normal((2900, nkv * hd)).astype(np.float32) for _ in range(2))
        k *= np.linspace(0.01, 3, 2900, dtype=np.float32)[:, None]
        k[[0, 5, 1000, 2899]] *= np.float32(20)
        m.write(0, 0, 0, k, v)
        m.reserve([2900], [2901])
        q, k, v = m.tokens(1)
        # scores reach 20 * 3 * 2 * 3: ten times those of TOL's bound, and so may be their errors
        _close(m.h.step(0, [2900], q, k, v), m.want(0, [2900], q, k, v), 10 * TOL)


# ---- the sparse step -----------------------------------------------------------


@pytest.mark.parametrize("cache", ["f32", "q8"])
@pytest.mark.parametrize("nh,nkv,hd", [(32, 8, 128), (32, 4, 64), (3, 1, 64), (6, 3, 128), (32, 2, 128)])
@pytest.mark.parametrize("pos,page_rows,keep", [
    ([0], 16, 1), ([40], 16, 1), ([40], 16, 2), ([255], 16, 7), ([256], 16, 16), ([256], 16, 17), ([700, 3, 1499, 64, 1000], 32, 9),
    ([1400, 15, 16], 16, 50), ([1000], 64, 100),
])
def test_sparse_step_matches_64_bits(nh, nkv, hd, pos, page_rows, keep, cache):
    m = Model(nh, nkv, hd, 1500, len(pos), cache, page_rows, bounds=True, key=sum(pos) + keep)
    with m.h:
        m.fill(pos)
        m.reserve(pos, [p + 1 for p in pos])
        q, k, v = m.tokens(len(pos))
        got, picked = m.h.step_sparse(0, pos, keep, q, k, v)
        want, pages = m.want_sparse(0, pos, keep, q, k, v)
        assert np.array_equal(picked, pages)
        _close(got, want)
        m.check_rows([p + 1 for p in pos])


def test_sparse_over_thousands_of_pages():
    """16000 pages of a sequence, the most there are."""
    m = Model(4, 2, 64, 16 * 16384, 1, "q8", 16, bounds=True, spare=0)
    with m.h:
        pos = 16 * 16000 + 5
        m.reserve([0], [pos + 1])
        # (values rise along the sequence by a little: keys in few groups, many equal scores)
        k = np.repeat(m.rng.standard_normal((40, 128)).astype(np.float32), 6401, axis=0)[:pos]
        v = m.rng.standard_normal((pos, 128)).astype(np.float32)
        m.h.write(0, 0, 0, k, v)
        at = np.arange(pos)
        m.p.rows[0, m.p.table[0, at // 16], 0, at % 16] = m.held(k)
        m.p.rows[0, m.p.table[0, at // 16], 1, at % 16] = m.held(v)
        for keep in (2, 100, 1500):
            q, kn, vn = m.tokens(1)
            got, picked = m.h.step_sparse(0, [pos], keep, q, kn, vn)
            want, pages = m.want_sparse(0, [pos], keep, q, kn, vn)
            assert np.array_equal(picked, pages)
            _close(got, want)


@pytest.mark.parametrize("cache", ["f32", "q8"])
def test_equal_scores_go_to_the_earlier_page(cache):
    m = Model(8, 2, 128, 2048, 2, cache, 16, bounds=True)
    with m.h:
        m.scatter([2000, 700])
        row = m.rng.standard_normal((1, 256)).astype(np.float32)
        for i, n in enumerate((2000, 700)):
            v = m.rng.standard_normal((n, 256)).astype(np.float32)
            m.write(i, 0, 0, np.repeat(row, n, axis=0), v)
        m.reserve([2000, 700], [2001, 701])
        q, k, v = m.tokens(2)
        got, picked = m.h.step_sparse(0, [2000, 700], 20, q, k, v)
        assert np.array_equal(picked[0, 0], list(range(19)) + [125])
        want, pages = m.want_sparse(0, [2000, 700], 20, q, k, v)
        assert np.array_equal(picked, pages)
        _close(got, want)


@pytest.mark.parametrize("cache", ["f32", "q8"])
def test_a_page_with_nan_is_picked_and_shows(cache):
    m = Model(8, 2, 128, 1024, 1, cache, 16, bounds=True)
    with m.h:
        m.fill([1000])
        row = np.full((1, 256), np.nan, np.float32)
        row[:, 128:] = 0
        m.h.write(0, 0, 500, row, None)
        m.reserve([1000], [1001])
        q, k, v = m.tokens(1)
        got, picked = m.h.step_sparse(0, [1000], 4, q, k, v)
        assert 500 // 16 in picked[0, 0] and np.isnan(got[0, :512]).all() and np.isfinite(got[0, 512:]).all()
        # a missing page too
        m.h.fork(None, [480])
        m.h.reserve([1000], [1001])
        got, picked = m.h.step_sparse(0, [1000], 4, q, k, v)
        assert picked[0, 0, :3].tolist() == [30, 31, 32] and np.isnan(got).all()


@pytest.mark.parametrize("cache", ["f32", "q8"])
@pytest.mark.parametrize("hd,page_rows", [(64, 16), (128, 16), (128, 64)])
def test_bounds_follow_what_is_written(hd, page_rows, cache):
    """By steps, row after row, over pages that held other rows, by writes, copies and compaction."""
    import torch
    top = 5 * page_rows
    m = Model(4, 2, hd, top, 3, cache, page_rows, bounds=True, layers=2)

    def check(lens):
        torch.cuda.synchronize()
        for l in range(2):
            at = m.h.view(l)["bounds"]

            class A:
                __cuda_array_interface__ = {"shape": (m.p.refs.size, 2, 2, hd), "typestr": "<f4", "data": (at, False), "version": 2}
            got = torch.as_tensor(A(), device="cuda").cpu().numpy()
            for i, n in enumerate(lens):
                for j in range(n // page_rows):
                    p = m.p.table[i, j]
                    keys = m.p.rows[l, p, 0].astype(np.float32).reshape(page_rows, 2, hd)
                    assert np.array_equal(got[p, :, 0], keys.min(axis=0)) and np.array_equal(got[p, :, 1], keys.max(axis=0))
    with m.h:
        m.reserve([0, 0, 0], [top, top, top])
        junk = np.full((top, 2 * hd), 9.0, np.float32)
        for i in range(3):
            for l in range(2):
                m.h.write(i, l, 0, junk, junk)
        m.fork(None, [0, 0, 0])
        pos = [0, 0, 0]
        m.fill([0, 21, 2 * page_rows])
        pos = [0, 21, 2 * page_rows]
        check(pos)
        for _ in range(2 * page_rows + 3):
            m.reserve(pos, [p + 1 for p in pos])
            for l in range(2):
                q, k, v = m.tokens(3)
                if l:
                    m.h.step(l, pos, q, k, v)
                else:
                    m.h.step_sparse(l, pos, 2, q, k, v)
                m.store(l, pos, k, v)
            pos = [p + 1 for p in pos]
        check(pos)
        rows = (m.rng.standard_normal((page_rows + 3, 2 * hd)) * 4).astype(np.float32)
        m.write(1, 1, 7, rows, rows)
        m.write(2, 0, page_rows - 1, rows[:1], rows[:1])
        check(pos)
        m.fork([1, 1, 0], pos[1:2] * 2 + pos[:1])
        pos = [pos[1], pos[1], pos[0]]
        m.reserve([3, 0, 0], [page_rows + 1, 0, 0])
        m.write(0, 0, 3, rows, rows)
        check(pos)
        m.fork(None, [pos[0], 0, pos[2]])
        pos[1] = 0
        assert m.h.compact() == m.p.compact()
        m.check_state()
        check(pos)


# ---- larger runs ------------------------------------------------------------------


@pytest.mark.parametrize("cache", ["f32", "q8"])
def test_pool_past_four_gibibytes(cache):
    """Pages whose byte offsets pass 2^32, and of a layer behind others."""
    nh, nkv, hd, R = 32, 32, 128, 128
    n_pages = (1 << 32) // (R * nkv * hd * (4 if cache == "f32" else 1)) + 40
    m = Model.__new__(Model)
    from tests import pages_model
    rng = rng_for(0x62696770)
    with PagedAttention(nh, nkv, hd, 4 * R, n_pages, R, n_layers=3, layer_begin=1, layer_end=3, max_batch=n_pages // 4 + 1, cache=cache,
                        bounds=True) as h:
        # the pool filled by others, the last pages for sequence 0
        others = n_pages // 4
        end = [0] + [4 * R] * others
        h.reserve([0] * (others + 1), end)
        table, _ = h.state()
        lastseq = others
        assert table[lastseq].max() >= n_pages - 5
        # the last sequence becomes sequence 0
        h.fork([lastseq], [4 * R])
        h.fork(list(range(1)) + [0] * others, [4 * R] + [0] * others)
        table, refs = h.state()
        assert refs.sum() == 4 and table[0].min() >= n_pages - 9
        pos = 3 * R + 17
        k, v = (rng.standard_normal((pos, nkv * hd)).astype(np.float32) for _ in range(2))
        h.write(0, 2, 0, k, v)
        from leap_amd.attention import HipAttention
        with HipAttention(nh, nkv, hd, 4 * R) as t:
            cos, sin = t.rope_download()
        from tests.helpers import attention_f64, rope_f32
        q, kn, vn = (rng.standard_normal((1, nkv * hd)).astype(np.float32) for _ in range(3))
        hold = lambda x: pages_model.held(x, hd, cache == "q8")  # noqa: E731
        K = np.concatenate([hold(k), hold(rope_f32(kn[0], cos[pos], sin[pos]))[None]])
        V = np.concatenate([hold(v), hold(vn)])
        m.hd, m.cos, m.sin = hd, cos, sin
        want = attention_f64(m.turned(q[0], pos), K, V, nh, nkv, hd)
        _close(h.step(2, [pos], q, kn, vn)[0], want)
        got, picked = h.step_sparse(2, [pos], 9, q, kn, vn)
        assert picked[0, 5].tolist() == [0, 1, 2, 3] + [-1] * 5
        _close(got[0], want)
        assert not h.read(0, 1, 0, R)[0].any()
        assert h.compact() == 4
        table, refs = h.state()
        assert sorted(table[0]) == [0, 1, 2, 3] and refs[:4].tolist() == [1] * 4
        _close(h.step(2, [pos], q, kn, vn)[0], want)


@pytest.mark.parametrize("cache", ["f32", "q8"])
def test_steps_on_a_stream_captured_and_replayed(cache):
    """Dense and sparse steps of two layers behind other work, replayed with other positions and tables."""
    import torch
    nh, nkv, hd = 32, 8, 128
    m = Model(nh, nkv, hd, 2048, 3, cache, 16, layers=2, bounds=True)
    with m.h:
        pos = [1500, 33, 700]
        m.fill(pos)
        m.reserve(pos, [p + 5 for p in pos])
        stream = torch.cuda.Stream()
        at, out, picked = _i32(pos), torch.zeros(2, 3, nh * hd, device="cuda"), _i32(np.zeros((3, nkv, 6)))
        d = [torch.zeros(2, 3, w, device="cuda") for w in (nh * hd, nkv * hd, nkv * hd)]

        def call():
            m.h.step_async(0, 3, _ptr(at), 1600, *[_ptr(x[0]) for x in d], _ptr(out[0]), stream.cuda_stream)
            m.h.step_sparse_async(1, 3, _ptr(at), 1600, 6, *[_ptr(x[1]) for x in d], _ptr(out[1]), _ptr(picked), stream.cuda_stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
        for step in range(4):
            tok = [m.tokens(3) for _ in range(2)]
            for l in range(2):
                for x, y in zip(d, tok[l]):
                    x[l].copy_(torch.from_numpy(y))
            at.copy_(_i32(pos))
            out.fill_(7.0)
            big = torch.randn(1024, 1024, device="cuda") @ torch.randn(1024, 1024, device="cuda")
            assert torch.isfinite(big).all()
            torch.cuda.synchronize()
            if step == 0:
                call()
            else:
                graph.replay()
            torch.cuda.synchronize()
            got = out.cpu().numpy()
            _close(got[0], m.want(0, pos, *tok[0]))
            want, pages = m.want_sparse(1, pos, 6, *tok[1])
            assert np.array_equal(picked.cpu().numpy(), pages)
            _close(got[1], want)
            pos = [p + 1 for p in pos]


def test_results_do_not_change_from_call_to_call():
    """The order in which runs arrive does not show."""
    import torch
    m = Model(32, 8, 128, 6000, 2, "f32", 32, bounds=True)
    with m.h:
        pos = [5900, 4000]
        m.fill(pos)
        m.reserve(pos, [p + 1 for p in pos])
        q, k, v = m.tokens(2)
        d, at = _dev(q, k, v), _i32(pos)
        outs = []
        for i in range(20):
            out = torch.empty(2, 32 * 128, device="cuda")
            if i % 2:
                m.h.step_sparse_async(0, 2, _ptr(at), 5999, 300, *map(_ptr, d), _ptr(out), 0, torch.cuda.current_stream().cuda_stream)
            else:
                m.h.step_async(0, 2, _ptr(at), 5999, *map(_ptr, d), _ptr(out), torch.cuda.current_stream().cuda_stream)
            outs.append(out)
        torch.cuda.synchronize()
        for i in range(2, 20):
            assert torch.equal(outs[i], outs[i % 2])


def test_rows_that_are_not_whole():
    m = Model(8, 2, 64, 64, 1)
    with m.h:
        m.reserve([0], [10])
        x = np.zeros(3 * 128, np.float32)
        for k, v in ((x[:-1], None), (x, x[:128]), (None, x[:5]), (x[:200], x[:200])):
            with pytest.raises(ValueError):
                m.h.write(0, 0, 0, k, v)
        m.h.write(0, 0, 0, x, x)


def test_refusals_of_a_handle():
    import torch
    m = Model(8, 2, 128, 64, 3, page_rows=16, layers=2)
    x = torch.zeros(8 * 128 * 3, device="cuda")
    p, i = x.data_ptr(), _i32([0, 0, 0])
    with m.h as h:
        z, zk = np.zeros((1, 1024), np.float32), np.zeros((1, 256), np.float32)
        _refused("layer", h.step, 2, [0], z, zk, zk)
        _refused("pos[0]", h.step, 0, [64], z, zk, zk)
        _refused("pos[0]", h.step, 0, [-1], z, zk, zk)
        _refused("n_seq", h.step_async, 0, 4, _ptr(i), 0, p, p, p, p)
        _refused("n_seq", h.step_async, 0, 0, _ptr(i), 0, p, p, p, p)
        _refused("max_pos", h.step_async, 0, 1, _ptr(i), 64, p, p, p, p)
        _refused("NULL", h.step_async, 0, 1, 0, 0, p, p, p, p)
        _refused("NULL", h.step_async, 0, 1, _ptr(i), 0, p, p, p, 0)
        _refused("aligned", h.step_async, 0, 1, _ptr(i), 0, p + 4, p, p, p)
        _refused("aligned", h.step_async, 0, 1, _ptr(i) + 2, 0, p, p, p, p)
        _refused("total_rows", h.step_async, 0, 1, _ptr(i), 9, p, p, p, p, 0, 11)
        _refused("bounds", h.step_sparse, 0, [0], 1, z, zk, zk)
        _refused("bounds", h.step_sparse_async, 0, 1, _ptr(i), 0, 1, p, p, p, p)
        _refused("rows [", h.reserve, [0, 5], [4, 4])
        _refused("rows [", h.reserve, [0], [65])
        _refused("rows [", h.reserve, [-1], [4])
        _refused("n_seq", h.reserve, [0] * 4, [1] * 4)
        _refused("n_seq", h.reserve, [], [])
        _refused("NULL", h.reserve_async, 1, 0, _ptr(i))
        _refused("aligned", h.reserve_async, 1, _ptr(i) + 1, _ptr(i))
        _refused("parent[0]", h.fork, [3], [0])
        _refused("parent[0]", h.fork, [-1], [0])
        _refused("rows[1]", h.fork, [0, 0], [0, 65])
        _refused("NULL", h.fork_async, 1, _ptr(i), 0)
        _refused("aligned", h.fork_async, 1, _ptr(i) + 2, _ptr(i))
        _refused("aligned", h.compact_async, _ptr(i) + 1)
        _refused("own", h.write, 0, 0, 0, zk, zk)
        _refused("position range", h.write, 0, 0, 64, zk, zk)
        _refused("seq", h.read, 3, 0, 0, 1)
        _refused("aligned", h.read_async, 0, 0, 0, 1, p + 4, 0)
        _refused("layer", h.view, 2)
        m.check_state()
        h.reserve([0, 0], [1, 1])
        h.fork([0, 0], [1, 1])
        _refused("own", h.write, 1, 0, 0, zk, zk)
    with PagedAttention(8, 2, 128, 64, 4, bounds=True) as h:
        _refused("keep", h.step_sparse, 0, [0], 0, z, zk, zk)
        _refused("keep", h.step_sparse_async, 0, 1, _ptr(i), 0, 0, p, p, p, p)
        _refused("aligned", h.step_sparse_async, 0, 1, _ptr(i), 0, 1, p, p, p, p, _ptr(i) + 2)


def test_a_create_that_does_not_fit_frees_everything():
    import torch
    free = torch.cuda.mem_get_info()[0]
    with pytest.raises(LeapError) as e:
        PagedAttention(32, 8, 128, 4096, 1 << 20, 128, n_layers=32)
    assert e.value.code == -errno.ENOMEM
    with PagedAttention(32, 8, 128, 4096, 10):
        pass
    assert torch.cuda.mem_get_info()[0] >= free - (64 << 20)


@pytest.mark.parametrize("cache", ["f32", "q8"])
@pytest.mark.parametrize("nh,nkv,hd,n_seq", [(32, 8, 128, 24), (8, 8, 128, 20), (64, 8, 128, 21), (32, 8, 64, 33), (8, 8, 64, 24), (128, 8, 64, 24),
                                             (16, 8, 64, 70)])
def test_unequal_batches(nh, nkv, hd, n_seq, cache):
    """Enough rows for a launch that shares the tiles out over the chip, and (70 sequences) too many sequences for it:
    lengths from one row on, positions out of range, shared and missing pages among them."""
    import torch
    m = Model(nh, nkv, hd, 1500, n_seq, cache, 16, key=n_seq)
    with m.h:
        pos = m.rng.integers(300, 1400, n_seq)
        pos[[0, 3, 5, 11, 12, 13]] = [0, 1, 15, 16, 1450, 63]
        pos[n_seq - 1] = 2
        m.fill(pos)
        m.fork(list(range(n_seq - 2)) + [4], [int(x) for x in pos[:-2]] + [20])   # the last but one shares a page with 4
        m.reserve(pos, [int(p) + 1 if i not in (6, n_seq - 2) else int(p) for i, p in enumerate(pos)])
        pos[n_seq - 2] = 7
        m.fork(None, [0 if i == 7 else int(p) + 1 for i, p in enumerate(pos)])    # 7 has no pages
        pos[8], pos[9] = -5, 1453
        m.reserve([0] * 6 + [int(pos[6])], [0] * 6 + [int(pos[6]) + 1])
        q, k, v = m.tokens(n_seq)
        d, out = _dev(q, k, v), torch.full((n_seq + 1, nh * hd), 3.0, device="cuda")
        at = _i32(pos)
        bad = [7, 8, 9, n_seq - 2]
        good = [i for i in range(n_seq) if i not in bad]
        # (the model stores the rows of those that are served)
        want = np.zeros((n_seq, nh * hd))
        for i in good:
            row = m.p.row(0, i, pos[i])
            row[0], row[1] = m.held(rope_f32(k[i], m.cos[pos[i]], m.sin[pos[i]])), m.held(v[i])
        for i in good:
            want[i] = attention_f64(m.turned(q[i], pos[i]), *m.p.of(0, i, int(pos[i]) + 1), nh, nkv, hd)
        for total in (0, int(np.maximum(pos, 0).sum()) + n_seq):
            out.fill_(3.0)
            m.h.step_async(0, n_seq, _ptr(at), 1450, *map(_ptr, d), _ptr(out), torch.cuda.current_stream().cuda_stream, total_rows=total)
            torch.cuda.synchronize()
            got = out.cpu().numpy()
            assert np.isnan(got[bad]).all() and (got[n_seq] == 3.0).all()
            _close(got[good], want[good])


@pytest.mark.parametrize("cache", ["f32", "q8"])
@pytest.mark.parametrize("nkv,pos,page_rows", [(1, [70000, 100, 30000, 65000, 0], 128), (2, [40000, 16, 33333], 64), (3, [30000, 29999, 1], 64),
                                               (8, [30000], 32)])
def test_unequal_batches_of_few_kv_heads(nkv, pos, page_rows, cache):
    """Fewer groups than XCDs, and one sequence far below the bound of its position."""
    import torch
    m = Model(4 * nkv, nkv, 64, 75000, len(pos), cache, page_rows, spare=0)
    with m.h:
        m.fill(pos)
        m.reserve(pos, [p + 1 for p in pos])
        q, k, v = m.tokens(len(pos))
        d, at = _dev(q, k, v), _i32(pos)
        want = m.want(0, pos, q, k, v)
        for total in (0, sum(pos) + len(pos)):
            out = torch.full((len(pos), 4 * nkv * 64), 3.0, device="cuda")
            m.h.step_async(0, len(pos), _ptr(at), 74999, *map(_ptr, d), _ptr(out), torch.cuda.current_stream().cuda_stream, total_rows=total)
            torch.cuda.synchronize()
            _close(out.cpu().numpy(), want)


@pytest.mark.parametrize("n_seq,rows", [(1100, 17), (3, 9000), (1024, 16), (1025, 16), (700, 30), (1024, 40)])
def test_more_pages_at_once_than_one_pass_takes(n_seq, rows):
    """Reservations of more than 1024 pages or sequences, missing and shared ones."""
    m = Model(1, 1, 64, rows + 16, n_seq, "q8", 16, spare=5, n_pages=n_seq * (rows // 16 + 1) + 30)
    with m.h:
        m.reserve([0] * n_seq, [rows - 1] * n_seq)
        m.check_state()
        parent = m.rng.integers(0, n_seq, n_seq).tolist()
        m.fork(parent, [rows - 1] * n_seq)
        m.check_state()
        last = m.rng.random(n_seq) < 0.9
        m.reserve([rows - 1 if x else 0 for x in last], [rows if x else 0 for x in last])
        m.check_state()
        begin = [0 if i < 900 else rows for i in range(n_seq)]
        m.reserve(begin, [rows] * n_seq)
        m.check_state()


@pytest.mark.parametrize("pages", [2048, 2049, 4096, 4097])
def test_sparse_around_a_threads_number_of_pages(pages):
    m = Model(2, 1, 64, 16 * 4200, 1, "f32", 16, bounds=True, spare=0, key=pages)
    with m.h:
        pos = 16 * pages + 3
        m.fill([pos])
        m.reserve([pos], [pos + 1])
        for keep in (2, 65, pages):
            q, k, v = m.tokens(1)
            got, picked = m.h.step_sparse(0, [pos], keep, q, k, v)
            want, chosen = m.want_sparse(0, [pos], keep, q, k, v)
            assert np.array_equal(picked, chosen)
            _close(got, want)


def test_two_graphs_of_a_handle_take_turns():
    """They share the handle's workspace; each replay leaves it as it was."""
    import torch
    nh, nkv, hd = 16, 4, 128
    m = Model(nh, nkv, hd, 3000, 12, "f32", 16, layers=1, bounds=True)
    with m.h:
        pos = [2900] + [700 + 130 * i for i in range(11)]
        m.fill(pos)
        m.reserve(pos, [p + 1 for p in pos])
        at = _i32(pos)
        tok = m.tokens(12)
        d = _dev(*tok)
        stream = torch.cuda.Stream()
        outs = [torch.zeros(12, nh * hd, device="cuda") for _ in range(3)]
        picked = _i32(np.zeros((12, nkv, 40)))

        def call(i):
            s = stream.cuda_stream
            if i == 0:
                m.h.step_async(0, 1, _ptr(at), 2999, *map(_ptr, d), _ptr(outs[0]), s)
            elif i == 1:
                m.h.step_async(0, 12, _ptr(at), 2999, *map(_ptr, d), _ptr(outs[1]), s)
            else:
                m.h.step_sparse_async(0, 12, _ptr(at), 2999, 40, *map(_ptr, d), _ptr(outs[2]), _ptr(picked), s)
        graphs = []
        torch.cuda.synchronize()
        for i in range(3):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                call(i)
        want = m.want(0, pos, *tok)
        sparse, pages = m.want_sparse(0, pos, 40, *tok)
        for i in (0, 1, 2, 1, 0, 2, 2, 0, 1, 1):
            for o in outs:
                o.zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                graphs[i].replay()
            torch.cuda.synchronize()
            if i == 2:
                assert np.array_equal(picked.cpu().numpy(), pages)
                _close(outs[2].cpu().numpy(), sparse)
            else:
                n = (1, 12)[i]
                _close(outs[i][:n].cpu().numpy(), want[:n])
                assert not outs[i][n:].any()


def test_two_handles_on_two_streams():
    import torch
    ms = [Model(32, 8, 128, 4096, 2, c, 32, key=i) for i, c in enumerate(("f32", "q8"))]
    try:
        jobs = []
        for m in ms:
            pos = [4000, 1234]
            m.fill(pos)
            m.reserve(pos, [p + 1 for p in pos])
            tok = m.tokens(2)
            jobs.append((m, pos, tok, _dev(*tok), _i32(pos), torch.zeros(8, 2, 32 * 128, device="cuda"), torch.cuda.Stream()))
        torch.cuda.synchronize()
        for i in range(8):
            for m, pos, tok, d, at, out, s in jobs:
                m.h.step_async(0, 2, _ptr(at), 4095, *map(_ptr, d), _ptr(out[i]), s.cuda_stream)
        torch.cuda.synchronize()
        for m, pos, tok, d, at, out, s in jobs:
            want = m.want(0, pos, *tok)
            for i in range(8):
                _close(out[i].cpu().numpy(), want)
    finally:
        for m in ms:
            m.h.close()
