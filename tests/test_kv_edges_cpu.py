"""The KV cache's C entry points on a host without a GPU, where sizes are at their edges."""
import ctypes as C

from dyn_quant import _lib
from test_kv_cpu import S3, append, attend, cache


def test_calls_beyond_the_grids_are_refused():
    c = cache()
    assert append(c, tokens=1 << 26) == _lib.DQ_ERR_UNSUPPORTED  # 2^27 rows
    assert append(c, tokens=2 ** 31 - 1) == _lib.DQ_ERR_UNSUPPORTED
    assert append(cache(kv_heads=65535), tokens=1025, ks=(0, 0, 128), vs=(0, 0, 128)) == _lib.DQ_ERR_UNSUPPORTED
    many = cache(n_seqs=1024)
    assert attend(many, tokens=1 << 20, q_heads=64) == _lib.DQ_ERR_UNSUPPORTED  # 2^36 rows in all
    assert _lib.lib().dq_kv_attend_workspace_bytes(C.byref(many), 1 << 20, 64, 0) == 0
    assert _lib.lib().dq_kv_attend_workspace_bytes(C.byref(many), 1 << 16, 64, 0) > 0
    assert attend(many, tokens=1 << 16, q_heads=64, q_stride=S3(0, 0, 128), ws_bytes=8) == _lib.DQ_ERR_WORKSPACE
