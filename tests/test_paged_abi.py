"""Refusals of the paged operators' C entries that need no GPU: NULL and
senseless arguments come back as an error that names the entry, and nothing is
touched."""
import ctypes

import pytest

from rustyllm_b200 import _lib

ENTRIES = ["rq_kv4_create", "rq_kv4_info", "rq_kv4_append", "rq_kv4_read", "rq_kv4_attention_workspace",
           "rq_kv4_attention", "rq_qk_norm_rope", "rq_qk_norm_rope_append", "rq_pages_extend", "rq_pages_release",
           "rq_spec_verify", "rq_llama_set_qk_norm", "rq_llama_use_kv4", "rq_llama_read_kv4"]


def nothing(t):
    return t(0) if issubclass(t, ctypes._SimpleCData) and t not in (ctypes.c_void_p, ctypes.c_char_p) else None


@pytest.mark.parametrize("name", ENTRIES)
def test_null_arguments_are_refused_by_name(name):
    f = getattr(_lib.lib(), name)
    assert f(*[nothing(t) for t in f.argtypes]) != 0
    assert name in _lib.last_error()


def test_attention_refuses_a_null_cache_before_its_query():
    q = _lib.Kv4Query()
    n = ctypes.c_size_t(7)
    assert _lib.lib().rq_kv4_attention_workspace(None, ctypes.byref(q), ctypes.byref(n)) != 0
    assert n.value == 7 and "rq_kv4_attention_workspace" in _lib.last_error()
    assert _lib.lib().rq_kv4_attention(None, ctypes.byref(q), None) != 0


def test_freeing_nothing_is_no_error():
    assert _lib.lib().rq_kv4_free(None) == 0
