"""The C++20 wrapper's cache of pages, through the demo's beam search."""
import os
import subprocess

import numpy as np
import pytest

from tests.conftest import gpu_available
from tests.helpers import attention_f64, rope_f32
from tests.test_gpu_beams import select

DEMO = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "leap_amd", "host", "engine_demo")
VOCAB = 1000
# (tests/test_gpu_pages.py derives the bound for scores of size 15; these are below 1)
TOL = 2e-5


def _run(*args):
    return subprocess.run([DEMO, *map(str, args)], capture_output=True, text=True, timeout=120)


def test_bad_beams_are_a_usage_error(tmp_path):
    for beams in (0, 17, -1):
        r = _run(2, 8, 2, 64, 16, 4, tmp_path, "pages", beams)
        assert r.returncode == 2 and "BEAMS" in r.stderr


def test_no_device_is_an_exception(tmp_path):
    if gpu_available():
        pytest.skip("a GPU is present")
    r = _run(2, 8, 2, 64, 16, 4, tmp_path, "pages", 4)
    assert r.returncode == 3 and "no HIP device" in r.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("nh,nkv,hd,beams,n_tok", [(16, 4, 128, 4, 50), (4, 4, 64, 1, 20), (8, 1, 64, 7, 40)])
def test_a_beam_search_of_the_engine(tmp_path, hip_device, nh, nkv, hd, beams, n_tok):
    from leap_amd.attention import HipAttention
    L, seq_len = 2, 64
    r = _run(L, nh, nkv, hd, seq_len, n_tok, tmp_path, "pages", beams)
    assert r.returncode == 0, r.stderr
    with HipAttention(nh, nkv, hd, seq_len) as t:
        cos, sin = t.rope_download()
    words = np.fromfile(tmp_path / "trace.bin", np.float32)
    sizes = [beams * n for n in (nh * hd, nkv * hd, nkv * hd, nh * hd)] * L + [beams * VOCAB] + [beams] * 3
    trace = words.reshape(n_tok, sum(sizes))
    rows = [[([], []) for _ in range(L)] for _ in range(beams)]
    score = np.full(beams, -np.inf, np.float32)
    score[0] = 0
    for pos in range(n_tok):
        parts = np.split(trace[pos], np.cumsum(sizes)[:-1])
        for layer in range(L):
            q, k, v, xb = (x.reshape(beams, -1) for x in parts[4 * layer:4 * layer + 4])
            for b in range(beams):
                K, V = rows[b][layer]
                K.append(rope_f32(k[b], cos[pos], sin[pos]))
                V.append(v[b])
                c, s = cos[pos].astype(np.float64), sin[pos].astype(np.float64)
                x = q[b].astype(np.float64).reshape(-1, hd)
                y = np.empty_like(x)
                y[:, 0::2], y[:, 1::2] = x[:, 0::2] * c - x[:, 1::2] * s, x[:, 1::2] * c + x[:, 0::2] * s
                want = attention_f64(y.reshape(-1), np.stack(K), np.stack(V), nh, nkv, hd)
                assert np.abs(xb[b] - want).max() <= TOL * np.abs(want).max()
        logits, best = parts[-4].reshape(beams, VOCAB), parts[-1]
        parent, token = parts[-3].view(np.int32), parts[-2].view(np.int32)
        wp, wt, wb = select(logits, score, 1, beams)
        assert parent.tolist() == list(wp) and token.tolist() == list(wt)
        # (logits below 8 and 1000 terms: sums in fp32, the logarithm in 64 bits, one rounding of a score below 1e3)
        assert np.abs(best - wb).max() <= 1e-6 * np.abs(wb).max() + 1e-5
        rows = [[(list(K), list(V)) for K, V in rows[p]] for p in parent]
        score = best.copy()
