"""The entry points of prompts, trees and the 8-bit cache without a device:
exported, declared in Python, and refusing a missing handle."""
import ctypes
import errno

import pytest

from leap_amd import attention


@pytest.fixture(scope="module")
def lib():
    return attention.load_library()


def test_a_missing_handle_is_refused(lib):
    i = ctypes.c_int
    args = (i * 4)()
    f = (ctypes.c_float * 4)()
    bad = -errno.EINVAL
    assert lib.leap_hip_attention_create_q8kv(None, None) == bad
    assert lib.leap_hip_attention_prompt(None, 0, 1, args, args, f, f, f, f) == bad
    assert lib.leap_hip_attention_tree(None, 0, 1, args, args, args, f, f, f, f) == bad
    assert lib.leap_hip_attention_tree_keep(None, 1, args, args, 1) == bad
    assert lib.leap_hip_attention_prompt_async(None, 0, 1, None, None, 1, 1, 1, None, None, None, None, None) == bad
    assert lib.leap_hip_attention_tree_async(None, 0, 1, None, None, None, 1, 1, 1, None, None, None, None, None) == bad
    assert lib.leap_hip_attention_tree_keep_async(None, 1, None, None, 1, None) == bad
    assert lib.leap_hip_attention_kv_write_async(None, 0, 0, 0, 1, None, None, None) == bad
    assert lib.leap_hip_attention_kv_read_async(None, 0, 0, 0, 1, None, None, None) == bad
    assert lib.leap_hip_attention_kv_q8_device_ptr(None, 0, 0, None, None, None, None) == bad


def test_create_refuses_what_the_fp32_create_refuses(lib):
    for change in ({"n_heads": 0}, {"n_kv_heads": 3}, {"head_dim": 96}, {"seq_len": 0}, {"max_batch": 0}):
        kw = dict(n_layers=1, layer_begin=0, layer_end=1, n_heads=8, n_kv_heads=2, head_dim=128, seq_len=64,
                  rope_theta=0.0, max_batch=1, device=0)
        kw.update(change)
        cfg, out = attention.Config(**kw), ctypes.c_void_p()
        assert lib.leap_hip_attention_create_q8kv(ctypes.byref(cfg), ctypes.byref(out)) == -errno.EINVAL
        assert not out.value


def test_an_unknown_cache_is_refused():
    with pytest.raises(ValueError):
        attention.HipAttention(8, 2, 128, 64, cache="f16")
