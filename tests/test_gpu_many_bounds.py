"""Prompts, trees and the 8-bit cache on inputs of very unlike magnitudes,
element by element against 64 bits, within bounds derived from what the header
states; each case asserts the kernel that it takes."""
import numpy as np
import pytest

from tests.helpers import rng_for, rope_f32
from tests.test_gpu_many import Model, _begin, _ptr
from tests.test_many_rules import plan

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _needs_gpu(hip_device):
    return hip_device


# The bound of one output element.  Elements of q, k and v are held to 2^-22 of
# themselves or 2^-34 of their row's largest.  Writing y for the rotated row of
# q, N_t for sum_i |y_i| |k_ti| / sqrt(hd) with every factor that is not 0
# raised by 2^-12 of its row's largest (2^-34 = 2^-22 * 2^-12):
#   a score is off by at most E = 2^-18 max N_t: 3 * 2^-22 for q, k and the
#     product of the low halves, under 2^-22 for the rotation, 8 * 2^-22 for
#     fp32 sums of 3 * 128 products in chains of at most 24 instructions,
#     3 * 2^-24 for its factors and the exponent: 16 * 2^-22 hold them all;
#   which moves an output by at most E sum_t p_t |v_t - out| (to first order,
#     E < 2^-6 here: 5% more), so by 2.1 E sum_t p_t |v_t| in any case;
#   values, probabilities, products and sums: 2^-20 sum_t p_t |v_t| (2^-22
#     twice, 2^-22 for the low halves, fp32 sums and the rounding of records);
#   values far below their row's largest m_t: 2^-34 sum_t p_t m_t;
#   weighted values p_t m_t far below the row of q's largest: each to 2^-30 of
#     that, and never by more than itself.
def reference(m, q, at, kr, vr, see, tight=False):
    """Outputs and bounds of the rows q (rotated at `at`) over the cache rows kr and vr [rows][kv_dim], see[row][cache row]."""
    nh, nkv, hd = m.nh, m.nkv, m.hd
    n, group = len(q), nh // nkv
    y = rotated(m, q.astype(np.float64), at).reshape(n, nh, hd)
    out, bound = np.empty((n, nh, hd)), np.empty((n, nh, hd))
    floor = lambda x: np.where(x == 0, 0, np.abs(x) + 2.0 ** -12 * np.abs(x).max(axis=1, keepdims=True))  # noqa: E731
    for h in range(nh):
        k, v = (x.reshape(-1, nkv, hd)[:, h // group] for x in (kr, vr))
        s = np.where(see, y[:, h] @ k.T / np.sqrt(hd), -np.inf)
        p = np.exp(s - s.max(axis=1, keepdims=True))
        p /= p.sum(axis=1, keepdims=True)
        out[:, h] = p @ v
        e = 2.0 ** -18 * np.where(see, floor(y[:, h]) @ floor(k).T / np.sqrt(hd), 0).max(axis=1, keepdims=True)
        assert e.max() < 2.0 ** -6
        mass = p @ np.abs(v)
        top = np.abs(v).max(axis=1)
        if tight:
            moved = 1.05 * np.stack([p[r] @ np.abs(v - out[r, h]) for r in range(n)])
        else:
            moved = 2.1 * mass
        bound[:, h] = (e * moved + 2.0 ** -20 * mass + 2.0 ** -34 * (p @ top)[:, None]
                       + np.minimum(p * top, see * 2.0 ** -30 * (p * top).max(axis=1, keepdims=True))
                       @ (np.abs(v) / np.maximum(top, 1e-300)[:, None]))
    return out.reshape(n, -1), bound.reshape(n, -1)


def rotated(m, x, at, back=False):
    """Rows of heads turned to their positions (back: from them), in 64 bits."""
    c, s = (np.repeat(t[at].astype(np.float64)[:, None], x.shape[1] // m.hd, axis=1) for t in (m.cos, m.sin))
    s = -s if back else s
    x = x.reshape(len(x), -1, m.hd)
    y = np.empty_like(x)
    y[..., 0::2], y[..., 1::2] = x[..., 0::2] * c - x[..., 1::2] * s, x[..., 1::2] * c + x[..., 0::2] * s
    return y.reshape(len(x), -1)


def within(got, want, bound):
    assert np.isfinite(got).all()
    worst = (np.abs(got - want) / np.maximum(bound, 1e-300)).max()
    assert worst <= 1, worst


class Run:
    """One sequence: `cached` rows, then n tokens as a prompt (or a step), with the caches' rows and q given."""

    def __init__(self, nh, nkv, hd, cache, cached, n, rows, step=False, key=0):
        assert plan(nh, nkv, hd, cache, (n,), (cached,), step).rows == rows
        self.m = Model(nh, nkv, hd, cached + n + 5, 1, cache, key=7919 * n + cached + key)
        self.cached, self.n, self.step = cached, n, step
        self.at = np.arange(cached, cached + n)
        self.see = np.arange(cached + n)[None] <= self.at[:, None]

    def out(self, y, k, v):
        """The call's outputs and the reference's for rotated queries y [n][q_dim] and the rows k and v of cache
        and tokens as they are to stand in the cache [cached + n][kv_dim], with the bound."""
        m, c = self.m, self.cached
        k, v = k.astype(np.float32), v.astype(np.float32)
        q = rotated(m, y, self.at, back=True).astype(np.float32)
        new = rotated(m, k[c:].astype(np.float64), self.at, back=True).astype(np.float32)
        if c:
            m.h.kv_upload(0, 0, 0, k[:c], v[:c])
        if self.step:
            got = m.h.step(0, c, q[0], new[0], v[c])[None]
        else:
            got = m.h.prompt(0, [0, self.n], [c], q, new, v[c:])
        kn = np.stack([rope_f32(new[j], m.cos[c + j], m.sin[c + j]) for j in range(self.n)])
        kr, vr = (np.concatenate([m.held(a), m.held(b)]) if c else m.held(b) for a, b in ((k[:c], kn), (v[:c], v[c:])))
        return got, q, kr, vr

    def check(self, y, k, v, rows=slice(None), tight=False):
        got, q, kr, vr = self.out(y, k, v)
        want, bound = reference(self.m, q[rows], self.at[rows], kr, vr, self.see[rows], tight)
        within(got[rows], want, bound)


# (heads, KV heads, head_dim, cache, cached rows, tokens, rows of a tile, a step)
KINDS = [
    (32, 8, 128, "f32", 500, 20, 16, False), (32, 4, 64, "f32", 700, 9, 16, False),
    (32, 8, 128, "f32", 500, 300, 256, False), (32, 8, 64, "f32", 300, 600, 256, False),
    (32, 8, 128, "q8", 900, 1, 16, True), (32, 4, 64, "q8", 333, 1, 16, True),
    (32, 8, 128, "q8", 500, 20, 16, False), (32, 8, 128, "q8", 300, 600, 256, False),
    (16, 4, 64, "q8", 300, 1700, 256, False),
]


def _directed(run, spread):
    """Queries along one direction of each KV head, and keys whose parts along it spread the scores by `spread`."""
    m, rng = run.m, run.m.rng
    T = run.cached + run.n
    u = rng.standard_normal((m.nkv, m.hd))
    u /= np.linalg.norm(u, axis=1, keepdims=True)
    b = 2.0 * np.sqrt(m.hd)
    y = np.repeat(b * u, m.nh // m.nkv, axis=0)[None] + 0.3 * rng.standard_normal((run.n, m.nh, m.hd))
    k = 0.3 * rng.standard_normal((T, m.nkv, m.hd))
    k -= (k * u).sum(axis=2, keepdims=True) * u
    score = spread * rng.standard_normal((T, m.nkv, 1))
    return y.reshape(run.n, -1), k, u, score, lambda s: (k + s * (np.sqrt(m.hd) / b) * u).reshape(T, -1)


@pytest.mark.parametrize("factor", [1e6, 1e10, 1e26])
@pytest.mark.parametrize("kind", KINDS)
def test_a_large_value_row_without_weight(kind, factor):
    """One visible value row larger than the rest by a factor, its score 60
    below them: next to nothing of it is in the outputs, and all of the rest."""
    run = Run(*kind, key=int(np.log10(factor)))
    with run.m.h:
        for where in (3, run.cached - 1):
            y, k, u, score, keys = _directed(run, 1.0)
            score[where] = -60.0
            v = run.m.rng.standard_normal((run.cached + run.n, run.m.nkv * run.m.hd))
            v[where] *= factor
            run.check(y, keys(score), v)


@pytest.mark.parametrize("order", ["mixed", "heavy last", "heavy first"])
@pytest.mark.parametrize("kind", KINDS)
def test_values_of_all_magnitudes_under_weights_of_all(kind, order):
    """Value rows from 1e-12 to 1e12 and scores over +-60: what outputs are
    made of is neither the heaviest nor the largest row."""
    run = Run(*kind, key=len(order))
    with run.m.h:
        y, k, u, score, keys = _directed(run, 20.0)
        T = run.cached + run.n
        if order != "mixed":
            score = np.sort(score, axis=0)[::1 if order == "heavy last" else -1]
        size = 10.0 ** run.m.rng.uniform(-12, 12, (T, 1))
        run.check(y, keys(score), size * run.m.rng.standard_normal((T, run.m.nkv * run.m.hd)))


@pytest.mark.parametrize("size", [1e38, 1e-28])
@pytest.mark.parametrize("kind", KINDS)
def test_values_at_the_ends_of_fp32(kind, size):
    """Values up to 3e38, whose weighted mean is finite, and near 1e-28."""
    run = Run(*kind, key=int(np.log10(size)) + 99)
    with run.m.h:
        y, k, u, score, keys = _directed(run, 1.0)
        shape = (run.cached + run.n, run.m.nkv * run.m.hd)
        run.check(y, keys(score), size * run.m.rng.uniform(1, 3, shape) * run.m.rng.choice([-1, 1], shape))

@pytest.mark.parametrize("what", ["values", "the first values", "every other value", "keys", "queries"])
@pytest.mark.parametrize("kind", KINDS)
def test_zeros(kind, what):
    """Rows of zeros, whose exponents mean nothing, alone and beside others."""
    run = Run(*kind, key=len(what))
    with run.m.h:
        m, T = run.m, run.cached + run.n
        y = 2.0 * m.rng.standard_normal((run.n, m.nh * m.hd))
        k, v = (m.rng.standard_normal((T, m.nkv * m.hd)) for _ in range(2))
        if what == "queries":
            y[:] = 0
        elif what == "keys":
            k[::3] = 0
        else:
            v[{"values": slice(None), "the first values": slice(0, run.cached), "every other value": slice(0, T, 2)}[what]] = 0
        run.check(y, k, v)


F32 = [k for k in KINDS if k[3] == "f32"]


@pytest.mark.parametrize("score", [30, 100])
@pytest.mark.parametrize("kind", F32)
def test_values_beside_a_larger_row(kind, score):
    """Three value rows with small elements beside one of 2^11 or 2^4 times
    their size that is masked: each element as exact as by itself.  (score: of
    a row's own key, which has nearly all the weight, or all that fp32 holds.)"""
    for ratio in (2.0 ** 11, 2.0 ** 3.9):
        run = Run(*kind, key=int(ratio))
        with run.m.h:
            m, T = run.m, run.cached + run.n
            k = m.rng.standard_normal((T, m.nkv, m.hd))
            v = m.rng.standard_normal((T, m.nkv, m.hd))
            first = [t for t in range((run.cached + 3) // 4 * 4, T - 4, max(4, run.n // 5 // 4 * 4))]
            y = np.zeros((run.n, m.nh, m.hd))
            rows = []
            for t in first:
                v[t:t + 3, :, m.hd // 4:] *= 1e-4
                v[t + 3] *= ratio
                for j in (t, t + 1, t + 2):
                    y[j - run.cached] = np.repeat(score / np.sqrt(m.hd) * k[j], m.nh // m.nkv, axis=0)
                    rows.append(j - run.cached)
            run.check(y.reshape(run.n, -1), k.reshape(T, -1), v.reshape(T, -1), rows, tight=True)


@pytest.mark.parametrize("kind", F32)
def test_keys_beside_a_larger_row(kind):
    """Scores that come from the small elements of three keys, beside a masked
    key of 2^11 times their size."""
    run = Run(*kind)
    with run.m.h:
        m, T = run.m, run.cached + run.n
        k = m.rng.standard_normal((T, m.nkv, m.hd))
        v = m.rng.standard_normal((T, m.nkv, m.hd))
        k[:, :, -2:] *= 2.0 ** -13
        first = [t for t in range((run.cached + 3) // 4 * 4, T - 4, max(4, run.n // 5 // 4 * 4))]
        y = np.zeros((run.n, m.nh, m.hd))
        rows = []
        for t in first:
            # the last pair of both: q 20 sqrt(hd) along that of the keys, which are alike
            k[t:t + 3, :, -2:] = k[t, :, -2:] * (1 + 0.01 * m.rng.standard_normal((3, m.nkv, 2)))
            k[t + 3] *= 2.0 ** 11
            k[t + 3, :, -2:] = 0  # (to later rows no more than others)
            for j in (t + 1, t + 2):
                pair = k[t, :, -2:]
                y[j - run.cached, :, -2:] = np.repeat(20 * np.sqrt(m.hd) * pair / (pair ** 2).sum(axis=1, keepdims=True),
                                                      m.nh // m.nkv, axis=0)
                rows.append(j - run.cached)
        run.check(y.reshape(run.n, -1), k.reshape(T, -1), v.reshape(T, -1), rows, tight=True)


@pytest.mark.parametrize("key,value,bad", [(1e-20, 1.0, 1e30), (2.0 ** -40, 1.0, 2.0 ** 126), (1.0, 2.0 ** -30, 2.0 ** 126)])
@pytest.mark.parametrize("kind", F32)
def test_small_rows_ahead_of_a_huge_masked_one(kind, key, value, bad):
    """Small keys under large queries, or small values, and a later token up to
    2^166 times as large in the same four positions."""
    run = Run(*kind, key=int(np.log2(bad)))
    with run.m.h:
        m, T = run.m, run.cached + run.n
        k, v = (x * m.rng.standard_normal((T, m.nkv * m.hd)) for x in (key, value))
        y = 2.0 / key * m.rng.standard_normal((run.n, m.nh * m.hd))
        late = T // 4 * 4 - 1
        (k if key != 1 else v)[late] = bad * m.rng.choice([-0.4, 0.4], m.nkv * m.hd)
        run.check(y, k, v, slice(0, late - run.cached))


@pytest.mark.parametrize("where,bad", [("k", 1e30), ("v", np.finfo(np.float32).max), ("k", np.nan), ("v", np.nan), ("v", np.inf)])
@pytest.mark.parametrize("kind", [k for k in KINDS if not k[7]])
def test_a_late_row_moves_nothing_ahead_of_it(kind, where, bad):
    """Huge elements, or one that is not finite, in a late token: every row
    ahead of it keeps its accuracy, and exactly the rows and heads that see a
    row that is not finite are NaN."""
    run = Run(*kind, key=17)
    with run.m.h:
        m, n = run.m, run.n
        late = n - 3
        y = 2.0 * m.rng.standard_normal((n, m.nh * m.hd))
        k, v = (m.rng.standard_normal((run.cached + n, m.nkv * m.hd)) for _ in range(2))
        if not np.isfinite(bad):
            {"k": k, "v": v}[where][run.cached + late, m.hd + 5] = bad  # KV head 1
            got, q, kr, vr = run.out(y, k, v)
            group = m.nh // m.nkv
            nan = np.isnan(got).reshape(n, m.nh, m.hd)
            want = np.zeros((n, m.nh, m.hd), bool)
            want[late:, group:2 * group] = True
            assert np.array_equal(nan, want)
        else:
            {"k": k, "v": v}[where][run.cached + late, 3::13] = bad
            got, q, kr, vr = run.out(y, k, v)
        rows = slice(0, late)
        kr, vr = (x[:run.cached + late] for x in (kr, vr))
        want, bound = reference(m, q[rows], run.at[rows], kr, vr, run.see[rows, :run.cached + late])
        within(got[rows], want, bound)

# Every form that a call is cut into, over both caches and in both head_dims:
# heads, KV heads, head_dim, new tokens and cached rows of the sequences, rows
# of a tile, one launch or two, more chunks than one, spread over the XCDs.
FORMS = [
    ("q8", 32, 8, 128, (8,), (300,), 16, True, False, False), ("f32", 3, 1, 64, (2,) * 100, (10,) * 100, 16, True, False, False),
    ("f32", 32, 8, 128, (33,), (30,), 16, False, False, False), ("q8", 32, 8, 128, (40,) * 9, (100,) * 9, 16, False, False, False),
    ("f32", 32, 8, 128, (8,), (300,), 16, True, True, False), ("q8", 32, 4, 64, (8,), (3000,), 16, True, True, False),
    ("f32", 3, 1, 64, (33,), (3000,), 16, False, True, False), ("q8", 32, 8, 128, (33,), (3000,), 16, False, True, False),
    ("f32", 3, 1, 64, (8,), (30000,), 16, True, True, True), ("q8", 8, 1, 128, (1,), (60000,), 16, True, True, True),
    ("f32", 32, 8, 128, (64,) * 40, (50,) * 40, 256, False, False, False), ("q8", 64, 8, 128, (700,), (0,), 256, False, False, False),
    ("f32", 8, 1, 128, (700,), (0,), 256, False, True, True), ("q8", 64, 8, 128, (64,) * 8, (1000,) * 8, 256, False, True, True),
    ("f32", 32, 4, 64, (64,), (12000,), 256, True, True, True), ("q8", 32, 8, 128, (64,) * 8, (2000,) * 8, 256, True, True, True),
    ("f32", 64, 4, 64, (33, 5, 64), (900, 2000, 0), 256, True, True, True),
]


@pytest.mark.parametrize("cache,nh,nkv,hd,lens,cached,rows,fused,split,spread,tree",
                         [f + (t,) for f in FORMS for t in (False, True) if not t or max(f[4]) <= 64])
def test_every_form_of_a_call(cache, nh, nkv, hd, lens, cached, rows, fused, split, spread, tree):
    p = plan(nh, nkv, hd, cache, lens, cached)
    assert (p.rows, p.fused, p.splits > 1, p.spread) == (rows, fused, split, spread), p
    m = Model(nh, nkv, hd, max(a + b for a, b in zip(lens, cached)), len(lens), cache, key=sum(lens) + tree)
    with m.h:
        for i, c in enumerate(cached):
            m.fill(i, c)
        begin = _begin(lens)
        parent = np.concatenate([[max(-1, j - int(m.rng.integers(1, 5))) for j in range(n)] for n in lens]).astype(np.int32)
        q, k, v = m.tokens(begin[-1])
        got = m.h.tree(0, begin, cached, parent, q, k, v) if tree else m.h.prompt(0, begin, cached, q, k, v)
        for i, (n, c) in enumerate(zip(lens, cached)):
            among = np.tril(np.ones((n, n), bool))
            if tree:
                among[:] = np.eye(n, dtype=bool)
                for j in range(n):
                    if parent[begin[i] + j] >= 0:
                        among[j] |= among[parent[begin[i] + j]]
            see = np.concatenate([np.ones((n, c), bool), among], axis=1)
            at = c + among.sum(axis=1) - 1
            for j in range(n):
                m.k[i, c + j] = m.held(rope_f32(k[begin[i] + j], m.cos[at[j]], m.sin[at[j]]))
                m.v[i, c + j] = m.held(v[begin[i] + j])
            rr = slice(begin[i], begin[i] + n)
            want, bound = reference(m, q[rr], at, m.k[i, :c + n], m.v[i, :c + n], see)
            within(got[rr], want, bound)
        m.check_cache([a + b for a, b in zip(lens, cached)])


# ---- bad nodes, bad bounds ---------------------------------------------------

# (heads, KV heads, head_dim, tokens, cached rows, rows of a tile, one launch)
TREES = [
    (8, 2, 128, (5,), (50,), 16, True), (32, 4, 64, (9, 3, 5), (7, 200, 0), 16, True),
    (8, 2, 128, (40, 5), (50, 3), 16, False), (32, 8, 128, (64,), (4000,), 256, True),
    (64, 8, 128, (40,), (4000,), 256, True), (32, 8, 128, (64,) * 9, (700,) * 9, 256, False),
]


@pytest.mark.parametrize("cache", ["f32", "q8"])
@pytest.mark.parametrize("nh,nkv,hd,lens,cached,rows,fused", TREES)
def test_what_is_stored_below_a_bad_node(nh, nkv, hd, lens, cached, rows, fused, cache):
    """A node whose parent is none counts as one on the cached rows for what is
    stored, and its descendants by their depth below it, in every form of call."""
    import torch
    got = plan(nh, nkv, hd, cache, lens, cached)
    if cache == "f32":
        assert (got.rows, got.fused) == (rows, fused), got
    m = Model(nh, nkv, hd, max(cached) + 70, len(lens), cache, key=sum(lens))
    with m.h:
        for i, c in enumerate(cached):
            m.fill(i, c)
        begin = _begin(lens)
        parent = np.concatenate([[j - 1 if j % 4 or not j else j - 3 for j in range(n)] for n in lens]).astype(np.int32)
        stored, bad = parent.copy(), np.zeros(len(parent), bool)
        for i, n in enumerate(lens):
            parent[begin[i] + n // 2] = (n // 2, -2, 77)[i % 3]  # itself, or no node at all
            stored[begin[i] + n // 2] = -1
            bad[begin[i] + n // 2] = True
            for j in range(n):
                if stored[begin[i] + j] >= 0:
                    bad[begin[i] + j] |= bad[begin[i] + stored[begin[i] + j]]
        assert bad.sum() > len(lens)
        q, k, v = m.tokens(begin[-1])
        want = m.want(begin, cached, q, k, v, stored)
        i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731
        d = [torch.from_numpy(x).cuda() for x in (q, k, v)]
        b, p, t = i32(begin), i32(cached), i32(parent)
        out = torch.full((len(q), nh * hd), 7.0, device="cuda")
        m.h.tree_async(0, len(lens), _ptr(b), _ptr(p), _ptr(t), len(q), max(lens), max(a + n - 1 for a, n in zip(cached, lens)),
                       *map(_ptr, d), _ptr(out), torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        got = out.cpu().numpy()
        assert np.isnan(got[bad]).all()
        assert np.abs(got[~bad] - want[~bad]).max() <= 1e-5 * np.abs(want[~bad]).max()
        m.check_cache([a + n for a, n in zip(cached, lens)])


def _nine_rows(cache):
    """Three sequences of 20 cached rows, nine rows of tokens on the device, a call and what the caches held."""
    import torch
    m = Model(8, 2, 128, 128, 3, cache)
    for i in range(3):
        m.fill(i, 20)
    before = [m.h.kv_download(i, 0, 0, 128) for i in range(3)]
    tokens = m.tokens(9)
    d = [torch.from_numpy(x).cuda() for x in tokens]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731

    def call(begin, max_tokens):
        out, b, p = torch.full((9, 1024), 7.0, device="cuda"), i32(begin), i32([20, 20, 20])
        m.h.prompt_async(0, 3, _ptr(b), _ptr(p), 9, max_tokens, 99, *map(_ptr, d), _ptr(out),
                         torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        return out.cpu().numpy()
    return m, tokens, before, call


def _untouched(m, i, before):
    after = m.h.kv_download(i, 0, 0, 128)
    assert np.array_equal(after[0], before[i][0]) and np.array_equal(after[1], before[i][1])


@pytest.mark.parametrize("cache", ["f32", "q8"])
def test_a_begin_ahead_of_the_arrays(cache):
    """A sequence whose rows begin below 0 comes back as NaN, the others are served."""
    m, (q, k, v), before, call = _nine_rows(cache)
    with m.h:
        got = call([-4, 3, 5, 8], 8)
        assert np.isnan(got[:3]).all() and (got[8:] == 7).all()
        want = m.want([3, 3, 5, 8], [20, 20, 20], q, k, v)
        assert np.abs(got[3:8] - want[3:8]).max() <= 1e-5 * np.abs(want[3:8]).max()
        _untouched(m, 0, before)


@pytest.mark.parametrize("cache", ["f32", "q8"])
def test_a_bound_of_no_tokens(cache):
    """Sequences with tokens under a bound of none come back as NaN."""
    m, _, before, call = _nine_rows(cache)
    with m.h:
        got = call([0, 2, 2, 5], 0)
        assert np.isnan(got[:5]).all() and (got[5:] == 7).all()
        for i in range(3):
            _untouched(m, i, before)


# ---- memory of transfers -----------------------------------------------------

def test_transfers_of_an_8_bit_cache_keep_little_memory():
    """A full slab up and down: the staging of fp32 rows stays a few MiB."""
    import torch
    rows, nkv, hd = 30000, 8, 128
    m = Model(8, nkv, hd, rows, 1, "q8")
    with m.h:
        k, v = (m.rng.standard_normal((rows, nkv * hd)).astype(np.float32) for _ in range(2))
        torch.cuda.synchronize()
        free = torch.cuda.mem_get_info()[0]
        m.h.kv_upload(0, 0, 0, k, v)
        a, b = m.h.kv_download(0, 0, 0, rows)
        assert free - torch.cuda.mem_get_info()[0] <= 64 << 20
        np.testing.assert_allclose(a, m.held(k), rtol=2.0 ** -24, atol=0)
        np.testing.assert_allclose(b, m.held(v), rtol=2.0 ** -24, atol=0)
        a, _ = m.h.kv_download(0, 0, 12345, 12350)
        np.testing.assert_allclose(a, m.held(k[12345:12350]), rtol=2.0 ** -24, atol=0)


@pytest.mark.parametrize("hd,cache", [(64, "f32"), (128, "f32"), (64, "q8")])
def test_keeping_a_path_allocates_nothing(hd, cache):
    """tree_keep_async behind a handle's first tree call, in a process of its
    own: the code it runs is on the device by then."""
    import subprocess
    import sys
    code = f"""
import torch
from leap_amd.attention import HipAttention
with HipAttention(8, 2, {hd}, 128, cache="{cache}") as h:
    x, kv = torch.zeros(4, {8 * hd}, device="cuda"), torch.zeros(4, {2 * hd}, device="cuda")
    b, z = torch.tensor([0, 4], dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    roots = z - 1
    s = torch.cuda.current_stream().cuda_stream
    h.tree_async(0, 1, b.data_ptr(), z.data_ptr(), roots.data_ptr(), 4, 4, 8, x.data_ptr(), kv.data_ptr(), kv.data_ptr(), x.data_ptr(), s)
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    h.tree_keep_async(1, z.data_ptr(), z.data_ptr(), 2, s)
    torch.cuda.synchronize()
    print("took", free - torch.cuda.mem_get_info()[0])
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "took 0\n" in r.stdout, r.stdout + r.stderr
