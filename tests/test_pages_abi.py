"""The entry points of caches of pages without a device: refusing a missing handle and bad configurations."""
import ctypes
import errno

import pytest

from leap_amd import attention as A
from tests.conftest import gpu_available


@pytest.fixture(scope="module")
def lib():
    return A.load_library()


def test_a_missing_handle_is_refused(lib):
    i, f, bad = (ctypes.c_int * 4)(), (ctypes.c_float * 4)(), -errno.EINVAL
    pages = lambda name, *args: getattr(lib, "leap_hip_attention_pages_" + name)(None, *args)  # noqa: E731
    assert pages("reserve", 1, i, i) == bad
    assert pages("reserve_async", 1, None, None, None, None) == bad
    assert pages("fork", 1, i, i) == bad
    assert pages("fork_async", 1, None, None, None) == bad
    assert pages("compact", i) == bad
    assert pages("compact_async", None, None) == bad
    assert pages("step", 0, 1, i, f, f, f, f) == bad
    assert pages("step_async", 0, 1, None, 0, 0, None, None, None, None, None) == bad
    assert pages("step_sparse", 0, 1, i, 1, f, f, f, f, i) == bad
    assert pages("step_sparse_async", 0, 1, None, 0, 1, None, None, None, None, None, None) == bad
    assert pages("write", 0, 0, 0, 1, f, f) == bad
    assert pages("write_async", 0, 0, 0, 1, None, None, None) == bad
    assert pages("read", 0, 0, 0, 1, f, f) == bad
    assert pages("read_async", 0, 0, 0, 1, None, None, None) == bad
    assert pages("clear") == bad
    assert pages("state", i, i) == bad
    assert pages("view", 0, None) == bad
    assert pages("beam_select", 1, 1, 4, f, f, i, i, f) == bad
    assert pages("beam_select_async", 1, 1, 4, None, 4, None, None, None, None, None) == bad
    assert pages("destroy") == 0
    assert lib.leap_hip_attention_pages_create(None, None) == bad


@pytest.mark.parametrize("change,fragment", [
    (dict(n_heads=0), "multiple"), (dict(n_kv_heads=3), "multiple"), (dict(head_dim=96), "head_dim"),
    (dict(n_heads=24, n_kv_heads=4), "head_dim"), (dict(n_heads=64, n_kv_heads=2), "head_dim"),
    (dict(seq_len=0), "seq_len"), (dict(seq_len=(1 << 24) + 1), "seq_len"), (dict(layer_end=2), "layer range"),
    (dict(max_batch=0), "max_batch"), (dict(max_batch=65536), "max_batch"), (dict(rope_theta=float("inf")), "rope_theta"),
    (dict(page_rows=0), "page_rows"), (dict(page_rows=8), "page_rows"), (dict(page_rows=48), "page_rows"),
    (dict(page_rows=256), "page_rows"), (dict(n_pages=0), "n_pages"), (dict(n_pages=(1 << 26) + 1), "n_pages"),
    (dict(q8=2), "q8"), (dict(bounds=-1), "bounds"), (dict(bounds=1, seq_len=16 * 16384 + 1), "pages a sequence"),
    (dict(n_heads=65536, n_kv_heads=65536, page_rows=16), "too large"),
    (dict(max_batch=2048, seq_len=1 << 24), "a table of 2048"), (dict(max_batch=65535, seq_len=1 << 24, page_rows=128), "a table of 65535"),
])
def test_create_refuses(lib, change, fragment):
    kw = dict(n_layers=1, layer_begin=0, layer_end=1, n_heads=8, n_kv_heads=2, head_dim=128, seq_len=64, rope_theta=0.0, max_batch=1,
              device=0, page_rows=16, n_pages=4, q8=0, bounds=0)
    kw.update(change)
    model = A.Config(*[kw[f] for f, _ in A.Config._fields_])
    cfg, out = A.PagesConfig(model, kw["page_rows"], kw["n_pages"], kw["q8"], kw["bounds"]), ctypes.c_void_p()
    assert lib.leap_hip_attention_pages_create(ctypes.byref(cfg), ctypes.byref(out)) == -errno.EINVAL
    assert not out.value
    assert fragment in lib.leap_hip_attention_pages_last_error(None).decode()


def test_create_without_a_device():
    if gpu_available():
        pytest.skip("a GPU is present")
    with pytest.raises(A.LeapError) as e:
        A.PagedAttention(8, 2, 128, 64, 4)
    assert e.value.code == -errno.ENODEV
    with pytest.raises(ValueError):
        A.PagedAttention(8, 2, 128, 64, 4, cache="f16")
