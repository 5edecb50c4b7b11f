"""What the attention entry points refuse before any device work (no GPU needed)."""
import ctypes as C

from diskmule_b200 import _native as N


def test_null_arguments():
    L = N.lib()
    bad = N.ERR_INVALID_ARGUMENT
    n, bits, h = C.c_uint64(), C.c_int32(), C.c_void_p()
    assert L.dm_attention_prompt(None, None, None) == bad
    assert L.dm_attention_status(None, None) == bad
    assert L.dm_kv_cache_create(None, None, C.byref(h)) == bad
    assert L.dm_kv_cache_describe(None, None) == bad
    assert L.dm_kv_cache_status(None, C.byref(bits), None) == bad
    for call in (L.dm_kv_cache_extend, L.dm_kv_cache_fork):
        assert call(None, None, None, 1, None) == bad
    assert L.dm_kv_cache_write(None, 0, None, None, None, None, None, None, 1, 1, None) == bad
    assert L.dm_kv_cache_compact(None, None, None, None, 1, 1, None) == bad
    assert L.dm_kv_cache_free(None, None, 1, None) == bad
    assert L.dm_kv_cache_copy_pages(None, None, None, 1, None) == bad
    assert L.dm_attention_decode_workspace(None, 1, 1, 0, 1, C.byref(n)) == bad
    assert L.dm_attention_decode(None, None, None) == bad
    assert b"null" in L.dm_last_error_message()
    L.dm_kv_cache_destroy(None)


def test_descriptors_match_the_header():
    """Sizes of the C structs on this ABI (LP64)."""
    assert C.sizeof(N.PromptDesc) == 8 * 4 + 2 * 8 + 5 * 8 + 8 * 8 + 2 * 8
    assert C.sizeof(N.KvCacheDesc) == 8 * 4 + 4 * 8
    assert C.sizeof(N.DecodeDesc) == 7 * 4 + 4 + 3 * 8 + 4 * 8 + 8 + 8 + 8
