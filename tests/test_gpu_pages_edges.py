"""Caches of pages at their edges: infinite keys head by head, and reservations of more than 1024 sequences or pages that
are refused in part or whole, in pools of more than 32768 pages."""
import errno

import numpy as np
import pytest

from leap_amd.attention import LeapError
from tests.helpers import attention_f64
from tests.pages_model import Model

pytestmark = pytest.mark.gpu

TOL = 2e-5  # (as for the step's other tests)


@pytest.fixture(scope="module", autouse=True)
def _needs_gpu(hip_device):
    return hip_device


def _ptr(t):
    return t.data_ptr()


def _i32(x):
    import torch
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def _cur():
    import torch
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("nh,nkv,hd,n_seq,pos,row", [(16, 4, 128, 2, 300, 123), (6, 2, 64, 1, 40, 0), (16, 2, 64, 1, 5000, 4999),
                                                     (32, 8, 128, 24, 1400, 700), (4, 1, 128, 1, 20000, 11111)])
@pytest.mark.parametrize("sign", [1, -1])
def test_an_infinite_key_head_by_head(nh, nkv, hd, n_seq, pos, row, sign):
    """One element of one key is infinite.  A q head whose rotated element has its sign has a score of +inf and a row of
    NaN; one whose element has the other sign has a score of -inf there and attends to the other rows."""
    m = Model(nh, nkv, hd, pos + 50, n_seq, "f32", 16, key=sign + 5)
    group, head, at = nh // nkv, nkv // 2, 7
    with m.h:
        lens = [pos - 3 * i for i in range(n_seq)]
        m.fill(lens)
        m.reserve(lens, [n + 1 for n in lens])
        x = m.p.row(0, 0, row)[0].astype(np.float32).copy()
        x[head * hd + at] = sign * np.inf
        m.h.write(0, 0, row, x[None], None)
        q, k, v = m.tokens(n_seq)
        want_sign = [sign if i % 2 == 0 else -sign for i in range(group)]
        y = m.turned(q[0], pos).reshape(nh, hd)
        for i in range(group):
            h = head * group + i
            if np.sign(y[h, at]) != want_sign[i]:
                q[0].reshape(nh, hd)[h] *= -1
        want = m.want(0, lens, q, k, v).reshape(n_seq, nh, hd)
        others = [r for r in range(pos + 1) if r != row]
        K, V = m.p.of(0, 0, others)
        without = attention_f64(m.turned(q[0], pos), K, V, nh, nkv, hd).reshape(nh, hd)
        got = m.h.step(0, lens, q, k, v).reshape(n_seq, nh, hd)
        for i in range(n_seq):
            for h in range(nh):
                expect = want[i, h]
                if i == 0 and h // group == head:
                    if want_sign[h % group] == sign:
                        assert np.isnan(got[0, h]).all(), h
                        continue
                    expect = without[h]
                assert np.isfinite(got[i, h]).all(), (i, h)
                assert np.abs(got[i, h] - expect).max() <= TOL * np.abs(want[i]).max(), (i, h)


@pytest.mark.parametrize("n_seq,rows", [(1100, 33), (40, 640)])
def test_a_large_reservation_that_does_not_fit(n_seq, rows):
    """More than 1024 sequences, or pages, that share pages, in a pool one page too small: nothing changes, twice over, and
    what is asked for afterwards goes as the rules say."""
    import torch
    width = (rows + 15) // 16
    n_pages = n_seq * width - 1
    m = Model(1, 1, 64, 16 * width, n_seq, "q8", 16, n_pages=n_pages)
    with m.h:
        m.fill([rows] + [0] * (n_seq - 1))
        m.fork([0] * n_seq, [rows] * n_seq)
        m.reserve([0] * (n_seq - 1), [1] * (n_seq - 1))     # the first pages of all but the last: copies
        m.check_state()
        # (for all rows of all sequences as their own it takes n_seq * width pages: the last who shares one keeps it)
        begin, end, status = _i32([0] * n_seq), _i32([rows] * n_seq), _i32([7] * n_seq)
        for _ in range(2):
            status.fill_(7)
            m.h.reserve_async(n_seq, _ptr(begin), _ptr(end), _ptr(status), _cur())
            torch.cuda.synchronize()
            assert not m.p.reserve([0] * n_seq, [rows] * n_seq)
            assert (status == -errno.ENOMEM).all()
            m.check_state()
        with pytest.raises(LeapError) as e:
            m.h.reserve([0] * n_seq, [rows] * n_seq)
        assert e.value.code == -errno.ENOMEM
        m.check_state()
        # some ask for the shared pages: by the short way and by the long one
        m.reserve([16] * 9, [32] * 9)
        m.check_state()
        half = [rows if i % 2 else 0 for i in range(n_seq)]
        m.reserve([0] * n_seq, half)
        m.check_state()
        lens = [rows] * n_seq
        m.check_rows(lens[:50])


def test_bad_ranges_among_many_sequences():
    import torch
    n_seq, top = 1100, 100
    m = Model(1, 1, 64, top, n_seq, "q8", 16, n_pages=n_seq * 7)
    with m.h:
        begin = m.rng.integers(0, top, n_seq)
        end = np.minimum(top, begin + m.rng.integers(0, 60, n_seq))
        bad = m.rng.random(n_seq) < 0.2
        bad[[0, n_seq - 1, 1023, 1024]] = True
        kinds = [(-1, 5), (5, 4), (0, top + 1), (-2147483648, 2147483647), (2147483647, 2147483647), (101, 101)]
        for i in np.flatnonzero(bad):
            begin[i], end[i] = kinds[i % len(kinds)]
        status = _i32([7] * n_seq)
        b, e = _i32(begin), _i32(end)
        m.h.reserve_async(n_seq, _ptr(b), _ptr(e), _ptr(status), _cur())
        torch.cuda.synchronize()
        assert np.array_equal(status.cpu().numpy(), np.where(bad, -errno.EINVAL, 0))
        assert m.p.reserve(np.where(bad, 0, begin).tolist(), np.where(bad, 0, end).tolist())
        m.check_state()
        # too few pages: the bad ones keep their own answer
        m2 = Model(1, 1, 64, top, n_seq, "q8", 16, n_pages=50)
        with m2.h:
            m2.h.reserve_async(n_seq, _ptr(b), _ptr(e), _ptr(status), _cur())
            torch.cuda.synchronize()
            assert np.array_equal(status.cpu().numpy(), np.where(bad, -errno.EINVAL, -errno.ENOMEM))
            m2.check_state()


def test_pools_of_more_pages_than_a_pass_lists():
    """Free and used pages are found 32768 at a time."""
    n_seq, width = 41, 1000
    m = Model(1, 1, 64, 16 * width, n_seq, "q8", 16, n_pages=40 * width + 7)
    lens = [16 * width] * 40 + [0]
    with m.h:
        m.reserve([0] * n_seq, lens)                       # the last pages lie behind 32768
        m.check_state()
        marks = {}
        for i in (0, 5, 33, 39):
            k, v = (m.rng.standard_normal((40, 64)).astype(np.float32) for _ in range(2))
            marks[i] = (k, v)
            m.write(i, 0, lens[i] - 40, k, v)
        m.reserve([0] * 41, [0] * 40 + [100])              # the last seven
        m.check_state()
        with pytest.raises(LeapError):
            m.h.reserve([0] * 41, [0] * 40 + [16 * 9])
        m.check_state()
        cut = [0 if i in (1, 2, 3, 34, 38) else 16 * 700 if i in (4, 35) else n for i, n in enumerate(lens[:40])] + [100]
        m.fork(None, cut)
        m.check_state()
        m.reserve([0] * 41, [0] * 40 + [16 * 600])         # pages before and behind
        m.check_state()
        used = m.p.compact()
        assert used > 32768 and m.h.compact() == used
        m.check_state()
        for i, (k, v) in marks.items():
            got = m.h.read(i, 0, lens[i] - 40, lens[i])
            for x, y in zip(got, (k, v)):
                np.testing.assert_allclose(x, m.held(y), rtol=2.0 ** -24, atol=0)
        m.fork(None, [0] * 20)
        used = m.p.compact()
        assert used < 32768 and m.h.compact() == used
        m.check_state()
