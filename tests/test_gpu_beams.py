"""The selection of a beam search, against its definition in 64 bits, and a search over a cache of pages."""
import errno

import numpy as np
import pytest

from leap_amd.attention import LeapError, PagedAttention
from tests.helpers import rng_for
from tests.pages_model import Model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _needs_gpu(hip_device):
    return hip_device


def _ptr(t):
    return t.data_ptr()


def select(logits, score, groups, beams):
    """The definition: totals in 64 bits; ties to the lower beam, the larger logit, the lower token."""
    vocab = logits.shape[1]
    parent, token, best = [], [], []
    for g in range(groups):
        rows, cand = range(g * beams, (g + 1) * beams), []
        for r in rows:
            x = logits[r].astype(np.float64)
            if np.isfinite(score[r]) and not np.isnan(x).any() and np.isfinite(x.max()):
                m = x.max()
                with np.errstate(divide="ignore"):
                    total = np.float64(score[r]) + x - (m + np.log(np.exp(x - m).sum()))
            else:
                total, x = np.full(vocab, -np.inf), np.zeros(vocab)
            at = np.lexsort((np.arange(vocab), -x))[:beams]
            cand += [(-total[t], r, -x[t], int(t)) for t in at]
        for total, r, _, t in sorted(cand)[:beams]:
            parent.append(r)
            token.append(t)
            best.append(-total)
    return np.array(parent), np.array(token), np.array(best)


def _check(got, logits, score, groups, beams):
    parent, token, best = select(logits, score, groups, beams)
    assert np.array_equal(got[0], parent) and np.array_equal(got[1], token)
    # a total is x - lse + score in 64 bits, lse by an fp32 sum of exponentials of fp32's exp2: terms of |x - max| up to
    # 40 are off by 40 log2(e) 2^-24 + 2^-22 and those that matter (|x - max| < 17) by half of that, sums over a wave
    # by 70 2^-24: under 6e-6 of lse at the worst; rounded once to fp32
    fin = np.isfinite(best)
    assert np.array_equal(np.isfinite(got[2]), fin) and (got[2][~fin] == -np.inf).all()
    assert (np.abs(got[2][fin] - best[fin]) <= 6e-6 + np.abs(best[fin]) * 2.0 ** -24).all()


@pytest.fixture(scope="module")
def h():
    with PagedAttention(8, 4, 64, 16, 1, max_batch=700) as h:
        yield h


@pytest.mark.parametrize("groups,beams,vocab", [
    (1, 1, 1), (1, 1, 2), (1, 4, 4), (1, 4, 5), (3, 5, 63), (2, 16, 16), (2, 16, 1000), (1, 4, 32000), (5, 3, 1023), (5, 3, 1024), (5, 3, 1025),
    (4, 8, 4097), (7, 2, 50257), (2, 8, 128256), (1, 16, 262144), (40, 16, 300), (233, 3, 999), (600, 1, 2500), (3, 4, 70001), (30, 8, 66000), (1, 2, 131072),
    (1, 2, 131073),
])
def test_selection_matches_64_bits(h, groups, beams, vocab):
    rng = rng_for(0x6265616D, groups, beams, vocab)
    n = groups * beams
    logits = (rng.standard_normal((n, vocab)) * 3).astype(np.float32)
    logits[rng.integers(0, n, 2 * n), rng.integers(0, vocab, 2 * n)] += np.float32(9)
    score = (-20 * rng.random(n)).astype(np.float32)
    _check(h.beam_select(groups, beams, logits, score), logits, score, groups, beams)


@pytest.mark.parametrize("beams,vocab", [(4, 50), (8, 5000), (16, 70000), (5, 200000)])
def test_equal_logits(h, beams, vocab):
    """All equal; a few values only; and in blocks, so that a lane has most of the largest."""
    rng = rng_for(0x74696573, beams, vocab)
    score = np.zeros(2 * beams, np.float32)
    score[beams:] = rng.integers(-2, 1, beams)
    few = rng.integers(0, 3, (2 * beams, vocab)).astype(np.float32)
    block = np.zeros((2 * beams, vocab), np.float32)
    block[:, vocab // 3:vocab // 3 + 2 * beams] = 5
    strided = np.zeros((2 * beams, vocab), np.float32)
    strided[:, 8::256] = 4 + np.arange(strided[:, 8::256].shape[1], dtype=np.float32)[::-1] / 128
    zeros = np.where(rng.random((2 * beams, vocab)) < 0.5, np.float32(0), np.float32(-0.0))
    for logits in (np.full((2 * beams, vocab), 1.5, np.float32), few, block, strided, zeros):
        _check(h.beam_select(2, beams, logits, score), logits, score, 2, beams)


@pytest.mark.parametrize("beams,vocab", [(1, 40), (4, 300), (5, 9000), (8, 40000), (3, 100000), (2, 150000)])
def test_masks_and_rows_that_are_not_distributions(h, beams, vocab):
    rng = rng_for(0x6D61736B, beams, vocab)
    n = 6 * beams
    logits = rng.standard_normal((n, vocab)).astype(np.float32)
    score = -rng.random(n).astype(np.float32)
    ninf = np.float32(-np.inf)
    logits[0:beams][rng.random((beams, vocab)) < 0.99] = ninf             # most tokens masked
    logits[beams:2 * beams] = ninf                                        # all masked but one of each (a beam that ended)
    logits[np.arange(beams, 2 * beams), rng.integers(0, vocab, beams)] = 0
    score[2 * beams + 1:3 * beams] = ninf                                 # a search's start
    logits[3 * beams] = np.nan                                            # rows without a distribution
    logits[3 * beams + beams // 2, 7] = np.inf
    logits[4 * beams:5 * beams] = ninf                                    # nothing at all
    score[5 * beams] = np.nan
    logits[5 * beams:, :] = np.finfo(np.float32).min                      # the type's lowest value for a mask
    logits[5 * beams:, vocab // 2] = 1
    _check(h.beam_select(6, beams, logits, score), logits, score, 6, beams)


@pytest.mark.parametrize("offset,pad", [(0, 0), (1, 0), (3, 5), (2, 1)])
def test_strides_alignment_streams_and_replays(h, offset, pad):
    """Rows that start anywhere, scores updated in place, on a stream, captured and replayed."""
    import torch
    groups, beams, vocab = 3, 4, 30001
    rng = rng_for(0x73747264, offset, pad)
    n, stride = groups * beams, vocab + pad
    buf = torch.full((offset + n * stride,), 1e30, device="cuda")
    rows = buf[offset:].view(n, stride)[:, :vocab]
    score = torch.zeros(n, device="cuda")
    parent, token = (torch.full((n + 1,), -5, dtype=torch.int32, device="cuda") for _ in range(2))
    s = torch.cuda.Stream()
    h.beam_select(1, 1, np.zeros((1, 4), np.float32), [0])  # (the workspace)

    def call():
        h.beam_select_async(groups, beams, vocab, buf.data_ptr() + 4 * offset, stride, _ptr(score), _ptr(parent), _ptr(token), _ptr(score),
                            s.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        call()
    for i in range(4):
        logits = (rng.standard_normal((n, vocab)) * 3).astype(np.float32)
        sc = (-5 * rng.random(n)).astype(np.float32)
        rows.copy_(torch.from_numpy(logits))
        score.copy_(torch.from_numpy(sc))
        torch.cuda.synchronize()
        if i == 0:
            call()
        else:
            graph.replay()
        torch.cuda.synchronize()
        _check([x.cpu().numpy()[:n] for x in (parent, token, score)], logits, sc, groups, beams)
        assert parent[n] == -5 and token[n] == -5


def test_refusals(h):
    import torch
    x = torch.zeros(4096, device="cuda")
    p = x.data_ptr()

    def refused(fragment, *args):
        with pytest.raises(LeapError) as e:
            h.beam_select_async(*args)
        assert e.value.code == -errno.EINVAL and fragment in str(e.value)
    refused("beams", 1, 0, 10, p, 10, p, p, p, p)
    refused("beams", 1, 17, 100, p, 100, p, p, p, p)
    refused("groups", 0, 1, 10, p, 10, p, p, p, p)
    refused("groups", 701, 1, 10, p, 10, p, p, p, p)
    refused("vocab", 1, 4, 3, p, 10, p, p, p, p)
    refused("vocab", 1, 4, 262145, p, 1 << 20, p, p, p, p)
    refused("stride", 1, 4, 10, p, 9, p, p, p, p)
    refused("NULL", 1, 4, 10, 0, 10, p, p, p, p)
    refused("NULL", 1, 4, 10, p, 10, p, 0, p, p)
    refused("aligned", 1, 4, 10, p + 2, 10, p, p, p, p)
    with PagedAttention(8, 4, 64, 16, 1, max_batch=4) as fresh:
        s = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            with pytest.raises(LeapError) as e:
                fresh.beam_select_async(1, 4, 10, p, 10, p, p, p, p, s.cuda_stream)
            x.add_(1)
        assert "captur" in str(e.value)


@pytest.mark.parametrize("cache", ["f32", "q8"])
def test_a_beam_search(cache):
    """A run of them together, all on the device: steps over pages, a toy model's logits, the selection, the fork by its
    parents and the next row's page, captured once and replayed for every token; against the same search on the model."""
    import torch
    nh, nkv, hd, groups, beams, vocab, prompt, steps = 8, 2, 64, 2, 3, 211, (21, 40), 40
    n = groups * beams
    m = Model(nh, nkv, hd, 128, n, cache, 16, layers=2)
    rng = rng_for(0x73656172)
    emb = [rng.standard_normal((vocab, w)).astype(np.float32) for w in (nh * hd, nkv * hd, nkv * hd)]
    # (logits far enough apart for the search to be the same in 64 bits)
    head = (rng.standard_normal((nh * hd, vocab)) * 0.4).astype(np.float32)
    with m.h:
        lens = [prompt[i // beams] for i in range(n)]
        m.fill([lens[i] if i % beams == 0 else 0 for i in range(n)])
        m.fork([i // beams * beams for i in range(n)], lens)
        m.reserve(lens, [x + 1 for x in lens])
        m.check_state()
        s = torch.cuda.Stream()
        dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        d_emb, d_head = [dev(x) for x in emb], dev(head)
        token, parent, status = i32([5] * n), i32([0] * n), i32([0] * n)
        score0 = [0.0 if i % beams == 0 else -np.inf for i in range(n)]
        score = torch.tensor(score0, device="cuda")
        pos, nxt, after = i32(lens), i32(lens), i32(lens)
        out = torch.zeros(2, n, nh * hd, device="cuda")
        rows = [[torch.zeros(n, x.shape[1], device="cuda") for x in d_emb] for _ in range(2)]
        logits = torch.zeros(n, vocab, device="cuda")
        m.h.beam_select(1, 1, np.zeros((1, 4), np.float32), [0])

        def token_pass():
            st = torch.cuda.current_stream().cuda_stream
            for l in range(2):
                for x, e in zip(rows[l], d_emb):
                    torch.index_select(e, 0, token, out=x)
                if l:
                    rows[1][0].add_(out[0])
                m.h.step_async(l, n, _ptr(pos), 127, *[_ptr(x) for x in rows[l]], _ptr(out[l]), st)
            torch.matmul(out[1], d_head, out=logits)
            m.h.beam_select_async(groups, beams, vocab, _ptr(logits), vocab, _ptr(score), _ptr(parent), _ptr(token), _ptr(score), st)
            nxt.copy_(pos + 1)
            after.copy_(pos + 2)
            m.h.fork_async(n, _ptr(parent), _ptr(nxt), st)
            m.h.reserve_async(n, _ptr(nxt), _ptr(after), _ptr(status), st)
            pos.copy_(nxt)
        torch.cuda.synchronize()
        keep = [x.clone() for x in (token, score, pos)]
        with torch.cuda.stream(s):  # (libraries load their code outside of the capture; on buffers of no consequence)
            torch.matmul(out[1], d_head, out=logits)
        torch.cuda.synchronize()
        for x, y in zip((token, score, pos), keep):
            x.copy_(y)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            token_pass()
        tok, sc, at = [5] * n, np.array(score0, np.float32), list(lens)
        for step in range(steps):
            graph.replay()
            torch.cuda.synchronize()
            assert status.tolist() == [0] * n
            x = None
            for l in range(2):
                q, k, v = (e[tok] for e in emb)
                x = m.want(l, at, q if x is None else (q + x).astype(np.float32), k, v)
            _check_run(out[1].cpu().numpy(), x)
            lg = logits.cpu().numpy()
            assert np.abs(lg - x @ head.astype(np.float64)).max() <= 1e-3 * np.abs(lg).max()
            # (the selection from the logits as they are: the search goes the same way)
            p, t, b = select(lg, sc, groups, beams)
            assert parent.tolist() == p.tolist() and token.tolist() == t.tolist()
            sc = score.cpu().numpy()
            assert np.abs(sc - b).max() <= 1e-5 * np.abs(b).max() + 6e-6
            tok, at = t.tolist(), [a + 1 for a in at]
            m.p.fork(p.tolist(), at)
            assert m.p.reserve(at, [a + 1 for a in at])
            m.check_state()
        m.check_rows(at)
        # beams share what they have in common
        _, refs = m.h.state()
        assert refs.max() > 1
        assert m.h.compact() == m.p.compact()
        m.check_state()
        m.check_rows(at)


def _check_run(got, want):
    # (two layers: the second one's queries carry the first one's error of 2e-5, and scores move by it times the keys)
    assert np.isfinite(got).all()
    assert np.abs(got - want).max() <= 4e-4 * np.abs(want).max()
