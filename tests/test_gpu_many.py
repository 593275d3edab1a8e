"""Prompts, trees of drafted tokens and the 8-bit cache, through the C ABI,
against a plain implementation in 64 bits (and each against the decode step,
token by token)."""
import errno

import numpy as np
import pytest

from leap_amd.attention import HipAttention, LeapError
from tests.helpers import attention_f64, rng_for, rope_f32

pytestmark = pytest.mark.gpu

# Outputs are weighted means of values: with |v| <= V their error is at most
# 2 V (largest error of a score) + V (terms of the sums).  A score of these
# inputs (|q . k| / sqrt(hd) <= 30) is a sum of up to 128 products held to
# 3 * 2^-22 each plus fp32 sums: under 30 * (3 * 2^-22 + 2^-21) < 4e-5 at the
# very worst and near 1e-6 as it comes; exp and the sums add a few 2^-24.
# 1e-5 of the largest output is asserted.
TOL = 1e-5


@pytest.fixture(scope="module", autouse=True)
def _needs_gpu(hip_device):
    return hip_device


def _ptr(t):
    return t.data_ptr()


class Model:
    """A handle and the same caches in float64."""

    def __init__(self, nh, nkv, hd, seq_len, n_seq, cache, layers=1, key=0):
        self.nh, self.nkv, self.hd, self.n_seq, self.cache = nh, nkv, hd, n_seq, cache
        self.h = HipAttention(nh, nkv, hd, seq_len, n_layers=layers, max_batch=n_seq, cache=cache)
        self.cos, self.sin = self.h.rope_download()
        self.rng = rng_for(0x6D616E79, nh, nkv, hd, seq_len, n_seq, key)
        self.k = np.zeros((n_seq, seq_len, nkv * hd), np.float64)
        self.v = np.zeros_like(self.k)

    def held(self, rows):
        """What the cache holds of fp32 rows."""
        if self.cache == "f32":
            return np.asarray(rows, np.float64)
        x = np.asarray(rows, np.float32).reshape(-1, self.hd)
        a = np.maximum(np.abs(x).max(axis=1, keepdims=True), np.float32(2.0 ** -100))
        q = np.rint(x * (np.float32(127) / a)).astype(np.float64)
        return (q * (a / np.float32(127)).astype(np.float64)).reshape(np.shape(rows))

    def fill(self, seq, rows):
        if not rows:
            return
        k = self.rng.standard_normal((rows, self.nkv * self.hd)).astype(np.float32)
        v = self.rng.standard_normal((rows, self.nkv * self.hd)).astype(np.float32)
        self.h.kv_upload(seq, 0, 0, k, v)
        self.k[seq, :rows], self.v[seq, :rows] = self.held(k), self.held(v)

    def tokens(self, n):
        f = lambda w, s: (s * self.rng.standard_normal((n, w))).astype(np.float32)  # noqa: E731
        return f(self.nh * self.hd, 2.0), f(self.nkv * self.hd, 1.0), f(self.nkv * self.hd, 1.0)

    def want(self, begin, pos, q, k, v, parent=None):
        """Outputs in 64 bits, the caches updated."""
        out = np.full((len(q), self.nh * self.hd), np.nan)
        for i in range(len(pos)):
            n = begin[i + 1] - begin[i]
            sees, depth = [], []
            for j in range(n):
                p = j - 1 if parent is None else parent[begin[i] + j]
                sees.append([j] if p < 0 else sees[p] + [j])
                depth.append(len(sees[j]) - 1)
            for j in range(n):
                r, at = begin[i] + j, pos[i] + depth[j]
                self.k[i, pos[i] + j] = self.held(rope_f32(k[r], self.cos[at], self.sin[at]))
                self.v[i, pos[i] + j] = self.held(v[r])
            for j in range(n):
                r, at = begin[i] + j, pos[i] + depth[j]
                c, s = self.cos[at].astype(np.float64), self.sin[at].astype(np.float64)
                x = q[r].astype(np.float64).reshape(-1, self.hd)
                y = np.empty_like(x)
                y[:, 0::2], y[:, 1::2] = x[:, 0::2] * c - x[:, 1::2] * s, x[:, 1::2] * c + x[:, 0::2] * s
                rows = list(range(pos[i])) + [pos[i] + m for m in sees[j]]
                out[r] = attention_f64(y.reshape(-1), self.k[i, rows], self.v[i, rows], self.nh, self.nkv, self.hd)
        return out

    def check_cache(self, rows):
        for i, n in enumerate(rows):
            k, v = self.h.kv_download(i, 0, 0, n)
            # (fp32: the rows as the step stores them; 8 bits: value * scale rounded once)
            np.testing.assert_allclose(k, self.k[i, :n], rtol=2.0 ** -24 if self.cache == "q8" else 0, atol=0)
            np.testing.assert_allclose(v, self.v[i, :n], rtol=2.0 ** -24 if self.cache == "q8" else 0, atol=0)


def _close(got, want):
    assert np.isfinite(got).all()
    e = np.abs(got - want).max() / np.abs(want).max()
    assert e <= TOL, e


def _begin(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


SHAPES = [(32, 8, 128), (32, 4, 64), (4, 4, 128), (3, 1, 64), (6, 3, 128), (32, 2, 128), (16, 2, 64)]


@pytest.mark.parametrize("cache", ["f32", "q8"])
@pytest.mark.parametrize("nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("lens,cached", [
    ([1], [0]), ([5], [0]), ([33], [0]), ([64], [1]), ([130], [97]),
    ([1, 0, 7, 40], [300, 5, 0, 31]), ([65, 1], [0, 129]),
])
def test_prompt_matches_64_bits(nh, nkv, hd, lens, cached, cache):
    m = Model(nh, nkv, hd, 512, len(lens), cache, key=sum(lens) * 1000 + sum(cached))
    with m.h:
        for i, n in enumerate(cached):
            m.fill(i, n)
        begin = _begin(lens)
        q, k, v = m.tokens(begin[-1])
        got = m.h.prompt(0, begin, cached, q, k, v)
        _close(got, m.want(begin, cached, q, k, v))
        m.check_cache([a + b for a, b in zip(lens, cached)])


@pytest.mark.parametrize("cache", ["f32", "q8"])
@pytest.mark.parametrize("nh,nkv,hd", [(32, 8, 128), (32, 4, 64), (4, 4, 128), (16, 1, 128)])
def test_long_prompt_over_a_long_cache(nh, nkv, hd, cache):
    """Many tiles and chunks: 700 tokens after 900 rows, and a second sequence."""
    m = Model(nh, nkv, hd, 2048, 2, cache)
    with m.h:
        m.fill(0, 900)
        m.fill(1, 3)
        begin = _begin([700, 211])
        q, k, v = m.tokens(begin[-1])
        got = m.h.prompt(0, begin, [900, 3], q, k, v)
        want = m.want(begin, [900, 3], q, k, v)
        _close(got, want)
        m.check_cache([1600, 214])


@pytest.mark.parametrize("cache", ["f32", "q8"])
@pytest.mark.parametrize("nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("lens,cached", [([1], [0]), ([8], [257]), ([64], [0]), ([64, 3, 31], [100, 511, 0]),
                                         ([17], [1500])])
def test_tree_matches_64_bits(nh, nkv, hd, lens, cached, cache):
    m = Model(nh, nkv, hd, 1600, len(lens), cache, key=sum(lens) * 1000 + sum(cached))
    with m.h:
        for i, n in enumerate(cached):
            m.fill(i, n)
        begin = _begin(lens)
        parent = np.concatenate([[int(m.rng.integers(max(-1, j - 6), j)) for j in range(n)] for n in lens]).astype(np.int32)
        q, k, v = m.tokens(begin[-1])
        got = m.h.tree(0, begin, cached, parent, q, k, v)
        _close(got, m.want(begin, cached, q, k, v, parent))
        m.check_cache([a + b for a, b in zip(lens, cached)])


def test_tree_of_a_chain_is_a_prompt():
    m = Model(32, 8, 128, 1024, 1, "f32")
    with m.h:
        m.fill(0, 500)
        q, k, v = m.tokens(64)
        a = m.h.prompt(0, [0, 64], [500], q, k, v)
        b = m.h.tree(0, [0, 64], [500], np.arange(64) - 1, q, k, v)
        assert np.array_equal(a, b) or np.abs(a - b).max() <= TOL * np.abs(a).max()


def test_tree_of_one_long_path_and_of_roots():
    """The deepest chain (64 ancestors) and the flattest tree (no ancestors)."""
    for parent in (np.arange(64) - 1, np.full(64, -1)):
        m = Model(8, 2, 128, 256, 1, "f32")
        with m.h:
            m.fill(0, 70)
            q, k, v = m.tokens(64)
            got = m.h.tree(0, [0, 64], [70], parent, q, k, v)
            _close(got, m.want([0, 64], [70], q, k, v, parent))


@pytest.mark.parametrize("nh,nkv,hd", SHAPES)
@pytest.mark.parametrize("pos", [[0], [31], [200], [1777], [0, 1, 64, 1000, 1999]])
def test_q8_step_matches_64_bits(nh, nkv, hd, pos):
    m = Model(nh, nkv, hd, 2048, len(pos), "q8", key=sum(pos))
    with m.h:
        for i, n in enumerate(pos):
            m.fill(i, n)
        q, k, v = m.tokens(len(pos))
        if len(pos) == 1:
            got = m.h.step(0, pos[0], q, k, v)[None]
        else:
            got = m.h.step_batched(0, pos, q, k, v)
        _close(got, m.want(list(range(len(pos) + 1)), pos, q, k, v))
        m.check_cache([p + 1 for p in pos])


@pytest.mark.parametrize("cache", ["f32", "q8"])
def test_a_conversation(cache):
    """A run of them together: a prompt, decode steps, a drafted tree, the
    accepted path kept, more steps; each against 64 bits over the rows that
    plain decoding would have."""
    layers = 2
    m = Model(32, 8, 128, 512, 2, cache, layers=layers)
    twin = HipAttention(32, 8, 128, 512, n_layers=layers, max_batch=2, cache=cache)
    with m.h, twin:
        begin = _begin([150, 37])
        q, k, v = m.tokens(begin[-1])
        for l in range(layers):
            got = m.h.prompt(l, begin, [0, 0], q, k, v)
        _close(got, m.want(begin, [0, 0], q, k, v))
        pos = [150, 37]
        for _ in range(3):
            q, k, v = m.tokens(2)
            for l in range(layers):
                got = m.h.step_batched(l, pos, q, k, v)
            _close(got, m.want([0, 1, 2], pos, q, k, v))
            pos = [p + 1 for p in pos]
        lens = [20, 9]
        begin = _begin(lens)
        parent = np.concatenate([[int(m.rng.integers(max(-1, j - 4), j)) for j in range(n)] for n in lens]).astype(np.int32)
        q, k, v = m.tokens(begin[-1])
        for l in range(layers):
            got = m.h.tree(l, begin, pos, parent, q, k, v)
        _close(got, m.want(begin, pos, q, k, v, parent))
        paths = np.full((2, 20), -1, np.int32)
        kept = []
        for i, n in enumerate(lens):
            node, path = n - 1, []
            while node >= 0:
                path.append(node)
                node = parent[begin[i] + node]
            path = path[::-1]
            paths[i, :len(path)] = path
            kept.append(len(path))
            for x in (m.k, m.v):
                x[i, pos[i]:pos[i] + len(path)] = x[i, [pos[i] + a for a in path]]
        m.h.tree_keep(pos, paths)
        for l in range(layers):
            for i in range(2):
                kk, vv = m.h.kv_download(i, l, 0, pos[i] + kept[i])
                tol = 2.0 ** -24 if cache == "q8" else 0
                np.testing.assert_allclose(kk, m.k[i, :pos[i] + kept[i]], rtol=tol, atol=0)
                np.testing.assert_allclose(vv, m.v[i, :pos[i] + kept[i]], rtol=tol, atol=0)
        pos = [p + n for p, n in zip(pos, kept)]
        q, k, v = m.tokens(2)
        for l in range(layers):
            got = m.h.step_batched(l, pos, q, k, v)
        _close(got, m.want([0, 1, 2], pos, q, k, v))


def test_prompt_is_the_decode_steps():
    """The framework's own decode step, token by token, on the same rows."""
    m = Model(32, 8, 128, 256, 1, "f32")
    with m.h, HipAttention(32, 8, 128, 256) as step:
        q, k, v = m.tokens(100)
        got = m.h.prompt(0, [0, 100], [0], q, k, v)
        want = np.stack([step.step(0, t, q[t], k[t], v[t]) for t in range(100)])
        assert np.abs(got - want).max() <= TOL * np.abs(want).max()
        a, b = m.h.kv_download(0, 0, 0, 100), step.kv_download(0, 0, 0, 100)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


@pytest.mark.parametrize("cache", ["f32", "q8"])
@pytest.mark.parametrize("where,bad", [("k", np.inf), ("v", np.nan), ("k", np.nan), ("v", -np.inf)])
def test_rows_with_infinities_reach_only_what_sees_them(where, bad, cache):
    """A key or value that is not finite at token 40 of a prompt, a stale row
    behind the sequence and an unseen node of a tree: NaN for the rows that
    see it, the others as without it."""
    m = Model(8, 2, 128, 256, 1, cache)
    with m.h:
        m.h.kv_upload(0, 0, 100, np.full((100, 256), bad, np.float32), np.full((100, 256), bad, np.float32))
        q, k, v = m.tokens(90)
        want = m.want([0, 90], [0], q, k, v)
        {"k": k, "v": v}[where][40, 128 + 77] = bad  # KV head 1
        got = m.h.prompt(0, [0, 90], [0], q, k, v)
        seen = np.zeros((90, 8), bool)
        seen[40:, 4:] = True
        got, want = got.reshape(90, 8, 128), want.reshape(90, 8, 128)
        assert np.isnan(got[seen]).all()
        _close(got[~seen], want[~seen])
    m = Model(8, 2, 128, 256, 1, cache)
    with m.h:
        m.fill(0, 70)
        parent = np.array([-1, 0, 0, 1, 2, 2, 5])
        q, k, v = m.tokens(7)
        want = m.want([0, 7], [70], q, k, v, parent).reshape(7, 8, 128)
        {"k": k, "v": v}[where][2, 5] = bad  # KV head 0 of node 2; nodes 2, 4, 5, 6 see it
        got = m.h.tree(0, [0, 7], [70], parent, q, k, v).reshape(7, 8, 128)
        seen = np.zeros((7, 8), bool)
        seen[[2, 4, 5, 6], :4] = True
        assert np.isnan(got[seen]).all()
        _close(got[~seen], want[~seen])


def test_a_query_with_nan_spoils_its_own_row():
    m = Model(8, 2, 64, 256, 1, "f32")
    with m.h:
        q, k, v = m.tokens(50)
        want = m.want([0, 50], [0], q, k, v).reshape(50, 8, 64)
        q[20, 64 * 3 + 9] = np.nan
        q[21, 64 * 5] = np.inf
        got = m.h.prompt(0, [0, 50], [0], q, k, v).reshape(50, 8, 64)
        seen = np.zeros((50, 8), bool)
        seen[20, 3] = seen[21, 5] = True
        assert np.isnan(got[seen]).all()
        _close(got[~seen], want[~seen])


@pytest.mark.parametrize("cache", ["f32", "q8"])
@pytest.mark.parametrize("kscale,vscale", [(1e-20, 1e20), (3e4, 1e-15), (1e-3, 1e5)])
def test_magnitudes_far_from_one(kscale, vscale, cache):
    """Keys and values far outside fp16's range, queries that bring the scores back."""
    m = Model(8, 2, 128, 256, 1, cache)
    with m.h:
        q, k, v = m.tokens(70)
        q, k, v = (q / np.float32(kscale)).astype(np.float32), k * np.float32(kscale), v * np.float32(vscale)
        got = m.h.prompt(0, [0, 70], [0], q, k, v)
        _close(got, m.want([0, 70], [0], q, k, v))


def test_values_of_unlike_rows():
    """Rows whose values differ by many powers of ten, under weights that make
    up for it: each output keeps the error of its own size."""
    m = Model(4, 1, 128, 512, 1, "f32")
    with m.h:
        q, k, v = m.tokens(300)
        v *= (10.0 ** m.rng.integers(-6, 4, (300, 1))).astype(np.float32)
        got = m.h.prompt(0, [0, 300], [0], q, k, v)
        want = m.want([0, 300], [0], q, k, v)
        size = np.abs(want).reshape(300, 4, 128).max(axis=2, keepdims=True)
        assert (np.abs(got - want).reshape(300, 4, 128) / size).max() <= 4 * TOL


def test_equal_scores_and_one_heavy_score():
    """All scores equal (a mean), and one score 80 above the rest (a copy)."""
    m = Model(8, 2, 128, 1024, 1, "f32")
    with m.h:
        q, k, v = m.tokens(600)
        got = m.h.prompt(0, [0, 600], [0], 0 * q, k, v)
        _close(got, m.want([0, 600], [0], 0 * q, k, v))
        got = m.h.prompt(0, [0, 600], [0], q * 60, k, v)
        want = m.want([0, 600], [0], q * 60, k, v)
        # (scores of up to 60 * 30: their rounding, 2e3 * 2^-21, moves weights by 1e-3 where two are near equal)
        assert np.abs(got - want).max() <= 4e-3 * np.abs(want).max()


def test_rows_behind_the_last_sequence_and_skipped_sequences():
    """The device form: rows outside [begin[0], begin[n]) stay as they were;
    sequences that break their bounds come back as NaN and leave the cache."""
    import torch
    for cache in ("f32", "q8"):
        m = Model(8, 2, 128, 256, 4, cache)
        with m.h:
            for i in range(4):
                m.fill(i, 50)
            before = [m.h.kv_download(i, 0, 0, 256) for i in range(4)]
            q, k, v = m.tokens(60)
            d = [torch.from_numpy(x).cuda() for x in (q, k, v)]
            out = torch.full((60, 1024), 7.0, device="cuda")
            begin = torch.tensor([3, 13, 23, 33, 43], dtype=torch.int32, device="cuda")
            pos = torch.tensor([50, 95, -1, 50], dtype=torch.int32, device="cuda")
            m.h.prompt_async(0, 4, _ptr(begin), _ptr(pos), 60, 20, 99, *map(_ptr, d), _ptr(out),
                             torch.cuda.current_stream().cuda_stream)
            torch.cuda.synchronize()
            got = out.cpu().numpy()
            want = m.want([3, 13, 23, 33, 43], [50, 0, 0, 50], q, k, v)
            _close(got[3:13], want[3:13])
            _close(got[33:43], want[33:43])
            assert np.isnan(got[13:33]).all()
            assert (got[:3] == 7).all() and (got[43:] == 7).all()
            for i in (1, 2):
                after = m.h.kv_download(i, 0, 0, 256)
                assert np.array_equal(after[0], before[i][0]) and np.array_equal(after[1], before[i][1])
            # begins that go back: what is ahead of them is served
            begin = torch.tensor([0, 10, 5, 40, 70], dtype=torch.int32, device="cuda")
            pos = torch.tensor([50, 50, 50, 50], dtype=torch.int32, device="cuda")
            out.fill_(7.0)
            m.h.prompt_async(0, 4, _ptr(begin), _ptr(pos), 60, 40, 99, *map(_ptr, d), _ptr(out),
                             torch.cuda.current_stream().cuda_stream)
            torch.cuda.synchronize()
            got = out.cpu().numpy()
            _close(got[:10], m.want([0, 10], [50], q, k, v)[:10])
            assert np.isnan(got[10:]).all()
            # a parent that is no earlier node
            parent = torch.tensor([-1, 0, 2, 2, 1] + [-1] * 55, dtype=torch.int32, device="cuda")
            begin = torch.tensor([0, 5, 5, 5, 5], dtype=torch.int32, device="cuda")
            out.fill_(7.0)
            m.h.tree_async(0, 4, _ptr(begin), _ptr(pos), _ptr(parent), 60, 5, 99, *map(_ptr, d), _ptr(out),
                           torch.cuda.current_stream().cuda_stream)
            torch.cuda.synchronize()
            got = out.cpu().numpy()
            assert np.isnan(got[2:4]).all() and np.isfinite(got[[0, 1, 4]]).all() and (got[5:] == 7).all()


def test_q8_batched_step_skips_bad_positions():
    import torch
    m = Model(8, 2, 128, 256, 3, "q8")
    with m.h:
        for i in range(3):
            m.fill(i, 50)
        q, k, v = m.tokens(3)
        d = [torch.from_numpy(x).cuda() for x in (q, k, v)]
        out = torch.zeros(3, 1024, device="cuda")
        pos = torch.tensor([50, 99, 50], dtype=torch.int32, device="cuda")
        m.h.step_batched_async(0, 3, _ptr(pos), 60, *map(_ptr, d), _ptr(out), torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        got = out.cpu().numpy()
        want = m.want([0, 1, 2, 3], [50, 50, 50], q, k, v)
        assert np.isnan(got[1]).all()
        _close(got[[0, 2]], want[[0, 2]])


@pytest.mark.parametrize("nkv,hd,rows", [(8, 128, 1), (8, 128, 333), (3, 64, 77), (1, 64, 5), (1, 128, 2)])
def test_rows_into_an_8_bit_cache_and_back(nkv, hd, rows):
    import torch
    rng = rng_for(0x71386B76, nkv, hd, rows)
    k = rng.standard_normal((rows, nkv * hd)).astype(np.float32)
    v = (1e-3 * rng.standard_normal((rows, nkv * hd))).astype(np.float32)
    v[0, :hd] = 0
    k[-1, -hd:] *= np.float32(1e-38)
    if rows > 2:
        k[1, 3] = np.nan
    m = Model(nkv, nkv, hd, 400, 2, "q8", layers=2)
    with m.h:
        s = torch.cuda.Stream()
        dk, dv = torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda()
        bk, bv = torch.empty_like(dk), torch.empty_like(dv)
        torch.cuda.synchronize()
        m.h.kv_write_async(1, 1, 17, 17 + rows, _ptr(dk), _ptr(dv), s.cuda_stream)
        m.h.kv_read_async(1, 1, 17, 17 + rows, _ptr(bk), _ptr(bv), s.cuda_stream)
        s.synchronize()
        wk, wv = m.held(k), m.held(v)
        if rows > 2:
            wk[1, :hd] = np.nan
        np.testing.assert_allclose(bk.cpu().numpy(), wk, rtol=2.0 ** -24, atol=0)
        np.testing.assert_allclose(bv.cpu().numpy(), wv, rtol=2.0 ** -24, atol=0)
        hk, hv = m.h.kv_download(1, 1, 17, 17 + rows)
        np.testing.assert_array_equal(hk, bk.cpu().numpy())
        np.testing.assert_array_equal(hv, bv.cpu().numpy())
        for seq, layer in ((0, 0), (0, 1), (1, 0)):
            assert not np.any(m.h.kv_download(seq, layer, 0, 400)[0])
        assert not np.any(m.h.kv_download(1, 1, 0, 17)[0]) and not np.any(m.h.kv_download(1, 1, 17 + rows, 400)[1])
        m.h.clear()
        assert not np.any(m.h.kv_download(1, 1, 0, 400)[0])


def test_rows_into_an_fp32_cache_and_back():
    import torch
    with HipAttention(8, 2, 128, 64) as h:
        a = torch.randn(10, 256, device="cuda")
        b = torch.empty_like(a)
        s = torch.cuda.current_stream().cuda_stream
        h.kv_write_async(0, 0, 5, 15, _ptr(a), 0, s)
        h.kv_read_async(0, 0, 5, 15, _ptr(b), 0, s)
        torch.cuda.synchronize()
        assert torch.equal(a, b)


def test_replayed_graph_matches_eager_calls():
    """A prompt, a tree, keeping its path and an 8-bit step captured once and
    replayed with other inputs in the same buffers."""
    import torch
    for cache in ("f32", "q8"):
        with HipAttention(32, 8, 128, 1024, max_batch=2, cache=cache) as h, \
                HipAttention(32, 8, 128, 1024, max_batch=2, cache=cache) as e:
            g = torch.Generator(device="cuda").manual_seed(5)
            i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
            begin, pos, tb, tp = i32([0, 200, 260]), i32([0, 0]), i32([0, 12, 20]), i32([200, 60])
            parent, path = i32([max(-1, j - 2) for j in range(12)] + [j - 1 for j in range(8)]), i32([[1, 3, 5], [0, 1, -1]])
            sp = i32([203, 62])
            bufs = [torch.empty(n, w, device="cuda") for n in (260, 20, 2) for w in (4096, 1024, 1024, 4096)]

            def calls(a, s):
                p = [_ptr(b) for b in bufs]
                a.prompt_async(0, 2, _ptr(begin), _ptr(pos), 260, 200, 300, *p[:4], s)
                a.tree_async(0, 2, _ptr(tb), _ptr(tp), _ptr(parent), 20, 12, 300, *p[4:8], s)
                a.tree_keep_async(2, _ptr(tp), _ptr(path), 3, s)
                a.step_batched_async(0, 2, _ptr(sp), 300, *p[8:], s)

            def draw():
                for i, b in enumerate(bufs):
                    if i % 4 != 3:
                        b.normal_(generator=g)
                    else:
                        b.fill_(float("nan"))
            draw()
            s = torch.cuda.Stream()
            torch.cuda.synchronize()
            calls(h, s.cuda_stream)
            calls(e, s.cuda_stream)
            s.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                calls(h, s.cuda_stream)
            for _ in range(4):
                draw()
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                got = [b.clone() for b in bufs[3::4]]
                for b in bufs[3::4]:
                    b.fill_(float("nan"))
                torch.cuda.synchronize()
                calls(e, s.cuda_stream)
                s.synchronize()
                for a, b in zip(got, bufs[3::4]):
                    assert torch.equal(a, b)
                for i in range(2):
                    a, b = h.kv_download(i, 0, 0, 300), e.kv_download(i, 0, 0, 300)
                    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_the_first_call_under_capture_is_refused():
    import torch
    with HipAttention(8, 2, 128, 64) as h:
        x = torch.zeros(4, 1024, device="cuda")
        i = torch.zeros(2, dtype=torch.int32, device="cuda")
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            x.add_(1.0)
            with pytest.raises(LeapError) as ei:
                h.prompt_async(0, 1, _ptr(i), _ptr(i), 4, 4, 8, _ptr(x), _ptr(x), _ptr(x), _ptr(x), s.cuda_stream)
        assert ei.value.code == -errno.EINVAL and "captur" in str(ei.value)


def _refused(fragment, f, *args):
    with pytest.raises(LeapError) as ei:
        f(*args)
    assert ei.value.code == -errno.EINVAL and fragment in str(ei.value), str(ei.value)


def test_refusals():
    with HipAttention(8, 2, 128, 64, n_layers=2, max_batch=2) as h, HipAttention(8, 2, 128, 64, cache="q8") as h8:
        p = 4096  # an aligned address that no refused call uses
        pr, tr = h.prompt_async, h.tree_async
        _refused("layer", pr, 2, 1, p, p, 4, 4, 8, p, p, p, p)
        _refused("n_seq", pr, 0, 3, p, p, 4, 4, 8, p, p, p, p)
        _refused("n_seq", pr, 0, 0, p, p, 4, 4, 8, p, p, p, p)
        _refused("n_tokens", pr, 0, 1, p, p, -1, 0, 8, p, p, p, p)
        _refused("max_tokens", pr, 0, 1, p, p, 4, 5, 8, p, p, p, p)
        _refused("max_tokens", pr, 0, 1, p, p, 4, -1, 8, p, p, p, p)
        _refused("max_tokens", pr, 0, 1, p, p, 40, 40, 8, p, p, p, p)
        _refused("max_pos", pr, 0, 1, p, p, 4, 4, 64, p, p, p, p)
        _refused("max_pos", pr, 0, 1, p, p, 4, 4, -1, p, p, p, p)
        _refused("NULL", pr, 0, 1, 0, p, 4, 4, 8, p, p, p, p)
        _refused("NULL", pr, 0, 1, p, p, 4, 4, 8, p, p, p, 0)
        _refused("aligned", pr, 0, 1, p, p, 4, 4, 8, p, p + 4, p, p)
        _refused("aligned", pr, 0, 1, p + 2, p, 4, 4, 8, p, p, p, p)
        _refused("NULL", tr, 0, 1, p, p, 0, 4, 4, 8, p, p, p, p)
        _refused("64 nodes", tr, 0, 1, p, p, p, 65, 65, 63, p, p, p, p)
        _refused("max_path", h.tree_keep_async, 1, p, p, 65)
        _refused("n_seq", h.tree_keep_async, 3, p, p, 4)
        _refused("NULL", h.tree_keep_async, 1, 0, p, 4)
        pr(0, 1, p, p, 0, 0, 8, 0, 0, 0, 0)  # no tokens: nothing to do
        h.tree_keep_async(1, 0, 0, 0)
        z = np.zeros((4, 1024), np.float32)
        zk = np.zeros((4, 256), np.float32)
        _refused("begin[0]", h.prompt, 0, [-1, 4], [0], z, zk, zk)
        _refused("below", h.prompt, 0, [0, 5, 4], [0, 0], z, zk, zk)
        _refused("positions", h.prompt, 0, [0, 4], [61], z, zk, zk)
        _refused("positions", h.prompt, 0, [0, 4], [-1], z, zk, zk)
        _refused("parent", h.tree, 0, [0, 4], [0], [-1, 1, 0, 0], z, zk, zk)
        _refused("parent", h.tree, 0, [0, 4], [0], [-1, -2, 0, 0], z, zk, zk)
        _refused("path", h.tree_keep, [0], [[1, 1]])
        _refused("path", h.tree_keep, [0], [[2, 1]])
        _refused("path", h.tree_keep, [60], [[0, 4]])
        _refused("position range", h.kv_write_async, 0, 0, 60, 65, p, p)
        _refused("seq", h.kv_read_async, 2, 0, 0, 4, p, p)
        _refused("aligned", h.kv_read_async, 0, 0, 0, 4, p + 8, p)
        _refused("fp32", h.kv_q8_device_ptr, 0, 0)
        _refused("8 bits", h8.kv_device_ptr, 0, 0)
        _refused("8 bits", h8.kv_fill_normal, 1, 1.0)
        _refused("8 bits", h8.floor_async, 1, 0, 1, 10, 11)
        _refused("set_split", h8.set_split, 64)
        _refused("set_products", h8.set_products, True)
        _refused("set_fold_helper", h8.set_fold_helper, 0)


def test_block_on_an_8_bit_cache():
    """The sub-block with the 8-bit cache against the one with the fp32 cache:
    the projections are the same, the attention differs by the cache's rounding
    alone, which the output's q8 step shows."""
    from tests.helpers import block_inputs
    nh, nkv, hd = 16, 4, 128
    rng = rng_for(0x626C6B38)
    x, rms, wq, wk, wv, wo = block_inputs(rng, nh * hd, nkv * hd)
    m = Model(nh, nkv, hd, 128, 1, "q8")
    with m.h, HipAttention(nh, nkv, hd, 128) as f:
        m.fill(0, 60)
        f.kv_upload(0, 0, 0, m.k[0, :60].astype(np.float32), m.v[0, :60].astype(np.float32))
        for h in (m.h, f):
            h.set_layer_weights(0, rms, wq, wk, wv, wo)
        a, b = m.h.block(0, 60, x), f.block(0, 60, x)
        kf, vf = f.kv_download(0, 0, 60, 61)
        k8, v8 = m.h.kv_download(0, 0, 60, 61)
        # (half a step of 1/127 of a head row's largest, and the fp32 rounding of the products)
        for got, want in ((k8, kf), (v8, vf)):
            step = np.abs(want).reshape(nkv, hd).max(axis=1, keepdims=True) / 127
            assert (np.abs(got - want).reshape(nkv, hd) <= 0.5001 * step).all()
        # the new row has at most all of a head's weight: one half step in v, and
        # the keys' half steps move weights by |q| sqrt(hd) / 254 relative at most
        assert np.abs(a - b).max() <= 0.05 * np.abs(b - x).max()


# (heads, KV heads, head_dim, cache, tokens): enough (token, head) rows for
# the tiles of 256, after which the tokens are few enough for those of 16
BOTH = [(32, 8, 128, "f32", 600), (32, 8, 128, "q8", 600), (32, 8, 64, "f32", 600), (16, 4, 64, "q8", 1700),
        (8, 2, 128, "f32", 90), (8, 2, 64, "q8", 90)]


@pytest.mark.parametrize("where,bad", [("k", 1e30), ("v", 1e30), ("v", np.finfo(np.float32).max), ("k", -1e25), ("v", np.nan)])
@pytest.mark.parametrize("nh,nkv,hd,cache,n", BOTH)
def test_huge_rows_that_are_masked_move_nothing(nh, nkv, hd, cache, n, where, bad):
    """Keys and values of later tokens, ten powers of ten and more above the
    rest: rows ahead of them, in the same tiles, keep their accuracy."""
    m = Model(nh, nkv, hd, 2048, 1, cache, key=n)
    with m.h:
        m.fill(0, 150)
        q, k, v = m.tokens(n)
        for t in (5, 37, 38, 70, n - 3):
            {"k": k, "v": v}[where][t, t % 7::13] = bad
        got = m.h.prompt(0, [0, n], [150], q, k, v)
        # (each stretch of tokens by itself: what is behind it cannot matter)
        clean = k.copy(), v.copy()
        for x in clean:
            x[np.isnan(x) | (np.abs(x) > 1e20)] = 0
        want = m.want([0, n], [150], q, *clean)
        _close(got[:5], want[:5])
        if where == "v" and np.isnan(bad):
            assert np.isnan(got[n - 3:]).any()
    m = Model(nh, nkv, hd, 2048, 8, cache, key=n + 1)
    with m.h:
        cached = [1900, 3, 700, 0, 33, 1500, 1800, 64]
        for i, c in enumerate(cached):
            m.fill(i, c)
        begin = _begin([64] * 8)
        parent = np.concatenate([[-1] + [int(m.rng.integers(max(-1, j - 9), j)) for j in range(1, 64)] for _ in range(8)])
        for i in range(8):  # node 20 of each tree is a leaf
            p = parent[64 * i:64 * i + 64]
            p[p == 20] = 19
        q, k, v = m.tokens(begin[-1])
        want = m.want(begin, cached, q, k, v, parent)
        {"k": k, "v": v}[where][20::64] = bad
        got = m.h.tree(0, begin, cached, parent, q, k, v)
        ok = np.ones(512, bool)
        ok[20::64] = False
        _close(got[ok], want[ok])


@pytest.mark.parametrize("nh,nkv,hd", [(32, 8, 128), (32, 8, 64)])
@pytest.mark.parametrize("spread", [1e4, 1e9, 1e14])
@pytest.mark.parametrize("n", [25, 700])
def test_keys_and_values_of_unlike_rows(nh, nkv, hd, spread, n):
    """Neighbouring rows that differ by `spread`, each by its own scale: rows
    that only see the small ones are as exact as those that see the large."""
    m = Model(nh, nkv, hd, 1024, 1, "f32", key=int(np.log10(spread)) + n)
    with m.h:
        q, k, v = m.tokens(n)
        k[1::2] *= np.float32(1e-3)
        v[n // 2::3] *= np.float32(spread)
        got = m.h.prompt(0, [0, n], [0], q, k, v)
        want = m.want([0, n], [0], q, k, v)
        _close(got[:n // 2], want[:n // 2])
        _close(got[n // 2:], want[n // 2:])


@pytest.mark.parametrize("cache", ["f32", "q8"])
def test_more_than_a_wave_of_sequences(cache):
    """130 sequences of 0 to 5 tokens, and one step of all of them, some skipped."""
    import torch
    n_seq = 130
    m = Model(8, 2, 64, 128, n_seq, cache)
    with m.h:
        lens = m.rng.integers(0, 6, n_seq)
        cached = m.rng.integers(0, 100, n_seq)
        for i, c in enumerate(cached):
            m.fill(i, int(c))
        begin = _begin(lens)
        q, k, v = m.tokens(begin[-1])
        got = m.h.prompt(0, begin, cached, q, k, v)
        _close(got, m.want(begin, cached, q, k, v))
        pos = (cached + lens).astype(np.int32)
        q, k, v = m.tokens(n_seq)
        want = m.want(np.arange(n_seq + 1), pos, q, k, v)
        pos[[0, 64, 129]] = [-1, 125, 128]
        d = [torch.from_numpy(x).cuda() for x in (q, k, v)]
        out = torch.zeros(n_seq, 512, device="cuda")
        dp = torch.from_numpy(pos).cuda()
        m.h.step_batched_async(0, n_seq, _ptr(dp), 110, *map(_ptr, d), _ptr(out), torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        got = out.cpu().numpy()
        assert np.isnan(got[[0, 64, 129]]).all()
        ok = np.ones(n_seq, bool)
        ok[[0, 64, 129]] = False
        _close(got[ok], want[ok])


@pytest.mark.parametrize("nh,nkv,hd,cache", [(32, 8, 128, "f32"), (64, 8, 128, "q8"), (64, 8, 64, "f32"), (64, 4, 64, "q8")])
def test_large_trees_over_a_long_cache(nh, nkv, hd, cache):
    """64 nodes after 4000 rows: one launch that stores the nodes, chunks on
    all XCDs; on a stream of its own, behind other work, captured and replayed."""
    import torch
    m = Model(nh, nkv, hd, 4096, 1, cache)
    with m.h:
        m.fill(0, 4000)
        parent = np.array([max(-1, j - 1 - j % 5) for j in range(64)], np.int32)
        q, k, v = m.tokens(64)
        want = m.want([0, 64], [4000], q, k, v, parent)
        i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731
        begin, pos, par = i32([0, 64]), i32([4000]), i32(parent)
        src = [torch.from_numpy(x).cuda() for x in (q, k, v)]
        d = [torch.zeros_like(x) for x in src]
        out = torch.full((64, nh * hd), 7.0, device="cuda")
        s = torch.cuda.Stream()
        torch.cuda.synchronize()

        def call():
            m.h.tree_async(0, 1, _ptr(begin), _ptr(pos), _ptr(par), 64, 64, 4095, *map(_ptr, d), _ptr(out), s.cuda_stream)
        with torch.cuda.stream(s):
            big = torch.randn(2048, 2048, device="cuda")
            for _ in range(4):
                big = big @ big * 1e-3
            for a, b in zip(d, src):
                a.copy_(b)
            call()
        s.synchronize()
        first = out.cpu().numpy()
        _close(first, want)
        m.check_cache([4064])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            call()
        for _ in range(3):
            out.fill_(7.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert np.array_equal(out.cpu().numpy(), first)


@pytest.mark.parametrize("cache", ["f32", "q8"])
def test_keeping_paths_on_the_device(cache):
    """Paths that end early, do not ascend, are no nodes or leave the cache."""
    import torch
    m = Model(6, 3, 64, 100, 6, cache, layers=2)
    with m.h:
        for i in range(6):
            for l in range(2):
                k = m.rng.standard_normal((100, 192)).astype(np.float32)
                m.h.kv_upload(i, l, 0, k, -k)
        before = [[m.h.kv_download(i, l, 0, 100) for l in range(2)] for i in range(6)]
        pos = [10, 10, 10, 97, -1, 99]
        path = [[0, 2, 5, 9], [3, 3, 4, 5], [1, 64, 65, 66], [1, 2, 3, 4], [0, 1, 2, 3], [0, -1, 5, 6]]
        kept = [4, 1, 1, 2, 0, 1]
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        dp, dx = i32(pos), i32(path)
        m.h.tree_keep_async(6, _ptr(dp), _ptr(dx), 4, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        for i in range(6):
            for l in range(2):
                for was, now in zip(before[i][l], m.h.kv_download(i, l, 0, 100)):
                    want = was.copy()
                    for t in range(kept[i]):
                        want[pos[i] + t] = was[pos[i] + path[i][t]]
                    assert np.array_equal(now, want)


def test_rows_past_two_gibibytes():
    """A layer slab of 2.9 GB, on a handle that holds the second of three
    layers: rows of zeros but for the last ones, whose byte offsets pass 2^31."""
    nh, hd, seq_len, real = 32, 128, 180000, 40
    rng = rng_for(0x32676962)
    with HipAttention(nh, nh, hd, seq_len, n_layers=3, layer_begin=1, layer_end=2) as h:
        cos, sin = h.rope_download()
        for n, pos, tree in ((3, seq_len - 3, False), (64, seq_len - 64, True)):
            h.clear()
            k0, v0 = (rng.standard_normal((real, nh * hd)).astype(np.float32) for _ in range(2))
            h.kv_upload(0, 1, pos - real, k0, v0)
            q, k, v = (s * rng.standard_normal((n, nh * hd)).astype(np.float32) for s in (4.0, 1.0, 1.0))
            q, k, v = (x.astype(np.float32) for x in (q, k, v))
            parent = np.full(n, -1, np.int32)
            got = h.tree(1, [0, n], [pos], parent, q, k, v) if tree else h.prompt(1, [0, n], [pos], q, k, v)
            want = np.zeros((n, nh, hd))
            for j in range(n):
                at = pos if tree else pos + j
                qr = rope_f32(q[j], cos[at], sin[at]).astype(np.float64).reshape(nh, hd)
                own = [j] if tree else list(range(j + 1))
                ks = np.concatenate([k0] + [rope_f32(k[t], cos[pos if tree else pos + t], sin[pos if tree else pos + t])[None]
                                            for t in own]).astype(np.float64).reshape(-1, nh, hd)
                vs = np.concatenate([v0] + [v[t][None] for t in own]).astype(np.float64).reshape(-1, nh, hd)
                s = np.einsum("hd,thd->ht", qr, ks) / np.sqrt(hd)
                w = np.exp(s - np.maximum(s.max(axis=1, keepdims=True), 0))
                zeros = (pos - real) * np.exp(-np.maximum(s.max(axis=1), 0))
                want[j] = np.einsum("ht,thd->hd", w, vs) / (w.sum(axis=1) + zeros)[:, None]
            _close(got, want.reshape(n, -1))
            kk, vv = h.kv_download(0, 1, pos, pos + n)
            assert np.array_equal(vv, v)
            assert not np.any(h.kv_download(0, 1, 0, 1000)[0]) and not np.any(h.kv_download(0, 1, pos - real - 1000, pos - real)[1])


@pytest.mark.parametrize("nh,nkv,hd,cache,n", [(32, 8, 128, "f32", 600), (32, 8, 64, "f32", 600), (32, 8, 128, "q8", 600)])
@pytest.mark.parametrize("where,bad", [("k", np.inf), ("k", np.nan), ("v", -np.inf)])
def test_infinities_in_tiles_of_many_rows(nh, nkv, hd, cache, n, where, bad):
    """One key or value of KV head 3 that is not finite at token 333, and a
    quad of unlike neighbours beside it."""
    m = Model(nh, nkv, hd, 1024, 1, cache, key=n + 7)
    with m.h:
        m.fill(0, 61)
        q, k, v = m.tokens(n)
        v[329:331] *= np.float32(1e-7)
        k[331] *= np.float32(1e-6)
        want = m.want([0, n], [61], q, k, v).reshape(n, nh, hd)
        {"k": k, "v": v}[where][333, 3 * hd + 11] = bad
        got = m.h.prompt(0, [0, n], [61], q, k, v).reshape(n, nh, hd)
        seen = np.zeros((n, nh), bool)
        group = nh // nkv
        seen[333:, 3 * group:4 * group] = True
        assert np.isnan(got[seen]).all()
        _close(got[~seen], want[~seen])
