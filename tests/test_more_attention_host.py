"""What the entry points around the paged cache refuse before any device work (no GPU needed)."""
import ctypes as C

import pytest

from diskmule_b200 import _native as N


def test_null_arguments():
    L, bad = N.lib(), N.ERR_INVALID_ARGUMENT
    n, h = C.c_uint64(), C.c_void_p()
    assert L.dm_attention_chunk_workspace(None, None, C.byref(n)) == bad
    assert L.dm_attention_chunk_workspace(None, C.byref(N.ChunkDesc()), None) == bad
    assert L.dm_attention_chunk(None, C.byref(N.ChunkDesc()), None) == bad
    assert L.dm_attention_weights(None, C.byref(N.WeightsDesc()), None) == bad
    assert L.dm_attention_rotate(None, None, None, C.byref(N.RotateDesc()), None) == bad
    assert L.dm_rope_create(None, C.byref(N.RopeDesc()), C.byref(h)) == bad
    assert L.dm_kv_cache_evict(None, C.byref(N.EvictDesc()), None) == bad
    assert L.dm_kv_cache_evict(None, None, None) == bad
    assert b"null" in L.dm_last_error_message()
    L.dm_rope_destroy(None)


def test_descriptors_match_the_header(tmp_path):
    """Sizes and the last members' places, from the header through a C compiler."""
    import os
    import shutil
    import subprocess
    gcc = shutil.which("gcc")
    if not gcc:
        pytest.skip("no C compiler")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pairs = [("dm_attention_chunk_desc", "workspace_bytes", N.ChunkDesc), ("dm_rope_desc", "pair_axes", N.RopeDesc),
             ("dm_attention_rotate_desc", "offsets", N.RotateDesc),
             ("dm_attention_weights_desc", "weights_stride", N.WeightsDesc), ("dm_kv_cache_evict_desc", "keep", N.EvictDesc)]
    body = "".join(f'printf("%zu %zu\\n", sizeof({t}), offsetof({t}, {m}));' for t, m, _ in pairs)
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "diskmule_attention.h"\nint main(void) {' + body + "return 0;}\n")
    exe = str(tmp_path / "sizes")
    subprocess.run([gcc, "-I", os.path.join(root, "include"), str(src), "-o", exe], check=True)
    lines = subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split("\n")
    for (t, m, s), line in zip(pairs, lines):
        assert [int(x) for x in line.split()] == [C.sizeof(s), getattr(s, m).offset], t


@pytest.mark.parametrize("which", ["rope", "cache"])
def test_rotate_refuses_what_is_closed(which):
    """A closed rotation is not "no rotation", a closed cache not "no cache"."""
    from diskmule_b200 import DmError
    from diskmule_b200.attention import KvCache, Rope, rotate

    class Context:
        handle = None

    closed = (Rope if which == "rope" else KvCache).__new__(Rope if which == "rope" else KvCache)
    closed._h = None
    given = dict(rope=None, cache=None)
    given[which] = closed
    with pytest.raises(DmError) as e:
        rotate(Context(), type=N.BF16, head_dim=64, tokens=0, **given)
    assert e.value.status == N.ERR_INVALID_ARGUMENT and "closed" in str(e.value)
