"""Sequences that lack a page ahead of their new row: a step writes nothing for them and gives NaN, dense or sparse, in
every kind of launch, until the page is there; against a plain model whose attention is in 64 bits."""
import numpy as np
import pytest

from tests.helpers import attention_f64, rng_for, rope_f32
from tests.pages_model import Model

pytestmark = pytest.mark.gpu

# As for the step's other tests: errors of scores, exp, weights and sums of these inputs are near 1e-6 as they come and
# under 4e-5 of the largest output if all of 40 roundings fell the same way; half of that is asserted.
TOL = 2e-5


@pytest.fixture(scope="module", autouse=True)
def _needs_gpu(hip_device):
    return hip_device


def _close(got, want):
    assert np.isfinite(got).all()
    e = np.abs(got - want).max() / np.abs(want).max()
    assert e <= TOL, e


def _bounds(m, layer):
    """The layer's bounds [page][kv_head][2][head_dim], or None."""
    import torch
    torch.cuda.synchronize()
    at = m.h.view(layer)["bounds"]
    if not at:
        return None

    class A:
        __cuda_array_interface__ = {"shape": (m.p.refs.size, m.nkv, 2, m.hd), "typestr": "<f4", "data": (at, False), "version": 2}
    return torch.as_tensor(A(), device="cuda").cpu().numpy()


def _held_rows(m):
    """All rows of all sequences in layer 0."""
    return [np.stack(m.h.read(i, 0, 0, m.seq_len)) for i in range(m.n_seq)]


def _served(m, i, pos):
    """Whether a step at pos has every page, and the new row's for its own."""
    at = m.p.table[i, :pos // m.p.R + 1]
    return bool((at >= 0).all()) and m.p.refs[at[-1]] == 1


def _step(m, pos, keep, tok):
    return m.h.step(0, pos, *tok) if keep is None else m.h.step_sparse(0, pos, keep, *tok)[0]


def _check(m, pos, keep=None):
    """A step of the sequences 0..len(pos)-1: outputs, rows and bounds."""
    tok = m.tokens(len(pos))
    rows, bounds = _held_rows(m), _bounds(m, 0)
    served = [_served(m, i, p) for i, p in enumerate(pos)]
    got = _step(m, pos, keep, tok)
    q, k, v = tok
    for i, p in enumerate(pos):
        if served[i]:
            continue
        assert np.isnan(got[i]).all(), i
    now = _held_rows(m)
    for i, p in enumerate(pos):
        for r in np.flatnonzero(~np.isclose(now[i], rows[i], rtol=0, atol=0, equal_nan=True).all(axis=(0, 2))):
            # (of the sequences that were served, the row of the position)
            assert any(served[j] and pos[j] == r and m.p.table[j, r // m.p.R] == m.p.table[i, r // m.p.R] for j in range(len(pos))), (i, r)
    if bounds is not None:
        changed = np.flatnonzero(~np.isclose(_bounds(m, 0), bounds, rtol=0, atol=0, equal_nan=True).all(axis=(1, 2, 3)))
        ends = {m.p.table[i, p // m.p.R] for i, p in enumerate(pos) if served[i] and p % m.p.R == m.p.R - 1}
        assert set(changed.tolist()) <= ends
    good = [i for i in range(len(pos)) if served[i]]
    if keep is None:
        for i in good:
            row = m.p.row(0, i, pos[i])
            row[0], row[1] = m.held(rope_f32(k[i], m.cos[pos[i]], m.sin[pos[i]])), m.held(v[i])
        for i in good:
            _close(got[i], attention_f64(m.turned(q[i], pos[i]), *m.p.of(0, i, pos[i] + 1), m.nh, m.nkv, m.hd))
    return got, good


@pytest.mark.parametrize("cache", ["f32", "q8"])
@pytest.mark.parametrize("nh,nkv,hd,page_rows", [(8, 2, 128, 16), (6, 3, 64, 32)])
@pytest.mark.parametrize("keep", [None, 1, 2, 100])
def test_an_earlier_missing_page(keep, nh, nkv, hd, page_rows, cache):
    """The new row's page is there and its own, one before it is not; the row is its page's last, so that the bounds would
    follow.  Then the page comes, and the step is served."""
    R = page_rows
    m = Model(nh, nkv, hd, 10 * R, 3, cache, R, bounds=True)
    with m.h:
        m.fill([3 * R - 1, 3 * R - 1, 5])
        m.fork(None, [3 * R - 1, R, 5])                      # 1: the first page alone
        m.reserve([0, 2 * R, 0], [3 * R, 3 * R, 6])          # and the third
        pos = [3 * R - 1, 3 * R - 1, 5]
        got, good = _check(m, pos, keep)
        assert good == [0, 2]
        m.reserve([0, R], [0, R + 1])                        # the second
        m.check_state()
        if keep is not None:  # (bounds of the pages as they are)
            for i, n in ((0, 3 * R - 1), (1, 3 * R - 1)):
                k, v = (m.rng.standard_normal((n, nkv * hd)).astype(np.float32) for _ in range(2))
                m.write(i, 0, 0, k, v)
            tok = m.tokens(3)
            got, picked = m.h.step_sparse(0, pos, keep, *tok)
            want, pages = m.want_sparse(0, pos, keep, *tok)
            assert np.array_equal(picked, pages)
            _close(got, want)
        else:
            got, good = _check(m, pos)
            assert good == [0, 1, 2]


@pytest.mark.parametrize("cache", ["f32", "q8"])
@pytest.mark.parametrize("nh,nkv,hd,n_seq,pos", [
    (32, 8, 128, 24, 1400),    # flat
    (16, 8, 64, 70, 300),      # one run a group
    (32, 8, 128, 3, 5000),     # runs of a group on one XCD
    (4, 1, 128, 2, 20000),     # on all
])
def test_holes_in_every_kind_of_launch(nh, nkv, hd, n_seq, pos, cache):
    """A hole in the first, a middle and the last page but one of a third of the sequences, filled from their ends."""
    m = Model(nh, nkv, hd, pos + 33, n_seq, cache, 16)
    with m.h:
        at = [pos - 37 * (i % 7) for i in range(n_seq)]
        m.scatter([0] * n_seq)
        where = {}
        begin, end = [0] * n_seq, [0] * n_seq
        for i in range(0, n_seq, 3):
            where[i] = [0, (at[i] // 16) // 2, at[i] // 16 - 1][(i // 3) % 3]
        for i in range(n_seq):
            end[i] = 16 * where[i] if i in where else at[i] + 1
        m.reserve(begin, end)
        m.reserve([16 * where[i] + 16 if i in where else 0 for i in range(n_seq)], [at[i] + 1 if i in where else 0 for i in range(n_seq)])
        m.check_state()
        for i in range(n_seq):
            for a, b in ((0, end[i]), (16 * where[i] + 16, at[i]) if i in where else (0, 0)):
                if b > a:
                    k, v = (m.rng.standard_normal((b - a, nkv * hd)).astype(np.float32) for _ in range(2))
                    m.write(i, 0, a, k, v)
        _, good = _check(m, at)
        assert good == [i for i in range(n_seq) if i not in where]
        m.reserve([16 * where[i] + 3 if i in where else 0 for i in range(n_seq)], [16 * where[i] + 16 if i in where else 0 for i in range(n_seq)])
        _, good = _check(m, at)
        assert good == list(range(n_seq))


@pytest.mark.parametrize("cache", ["f32", "q8"])
@pytest.mark.parametrize("seed", range(4))
def test_steps_among_any_calls(seed, cache):
    """Reservations with gaps, forks of sequences with gaps, cuts, pools that are too small, compactions and clears in any
    order, and a step after each."""
    rng = rng_for(0x686F6C65, seed)
    R, n_seq, top = (16, 32)[seed % 2], 6, 240
    m = Model(4, 2, 64, top, n_seq, cache, R, bounds=seed >= 2, key=seed, n_pages=(60, 33)[seed % 2])
    served = missed = 0
    with m.h:
        for _ in range(60):
            n = int(rng.integers(1, n_seq + 1))
            what = rng.choice(["reserve", "reserve", "reserve", "fork", "cut", "compact"])
            if what == "reserve":
                begin = rng.integers(0, top, n).tolist()
                end = [min(top, b + int(rng.choice([0, 1, 20, 60, 120]))) for b in begin]
                if rng.random() < 0.6:
                    begin = [0] * n
                if m.p.reserve(begin, end):
                    m.h.reserve(begin, end)
                else:
                    with pytest.raises(Exception):
                        m.h.reserve(begin, end)
            elif what == "compact":
                assert m.h.compact() == m.p.compact()
            else:
                m.fork(None if what == "cut" else rng.integers(0, n_seq, n).tolist(), rng.integers(0, top + 1, n).tolist())
            m.check_state()
            pos = []
            for i in range(n_seq):
                there = np.flatnonzero(m.p.table[i] >= 0)
                j = int(rng.choice(there)) if there.size else int(rng.integers(0, top // R))
                pos.append(min(top - 1, j * R + int(rng.integers(0, R))))
            _, good = _check(m, pos)
            served += len(good)
            missed += n_seq - len(good)
        assert served > 40 and missed > 40
        m.h.clear()
        m.p.table[:], m.p.refs[:], m.p.rows[:] = -1, 0, 0
        m.reserve([0] * n_seq, [1] * n_seq)
        _check(m, [0] * n_seq)


@pytest.mark.parametrize("n_seq,rows", [(1100, 65), (60, 500)])
def test_holes_among_many_pages_at_once(n_seq, rows):
    """Reservations of more than 1024 sequences or pages that leave holes, and that fill them ahead of long runs."""
    m = Model(1, 1, 64, rows + 16, n_seq, "q8", 16, spare=5)
    with m.h:
        last = rows - 1
        some = m.rng.random(n_seq) < 0.5
        m.reserve([32 if x else 0 for x in some], [rows] * n_seq)
        m.check_state()
        _, good = _check(m, [last] * n_seq)
        assert good == np.flatnonzero(~some).tolist()
        m.reserve([0] * n_seq, [17 if x else 0 for x in some])
        _, good = _check(m, [last] * n_seq)
        assert len(good) == n_seq
