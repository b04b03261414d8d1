"""The KV cache's C entry points on a host without a GPU: sizes, and arguments
refused before any CUDA call; the Python class's own checks."""
import ctypes as C

import pytest

from dyn_quant import _lib
from dyn_quant.kv_cache import Int4KVCache, unit_bytes

P = C.c_void_p
S3 = C.c_int64 * 3


def cache(**kw):
    v = dict(units=256, mass=256, pos=256, lengths=256, evicted=256, page_table=256, arrivals=256, n_seqs=2, n_pages=8,
             max_pages=4, page_size=64, kv_heads=2, head_dim=128)
    v.update(kw)
    return _lib.DqKvCache(**v)


def append(c, k=256, v=256, ks=(1024, 256, 128), vs=(1024, 256, 128), tokens=4, counts=None, at=None, kv=None, vv=None):
    return _lib.lib().dq_kv_append(C.byref(c) if c else None, P(k), S3(*ks), P(v), S3(*vs), tokens, P(counts), P(at),
                                   P(kv), P(vv), None)


def attend(c, ws=256, ws_bytes=1 << 40, **kw):
    v = dict(q=256, q_stride=S3(1024, 1024, 128), out=256, out_stride=S3(1024, 1024, 128), lse=None, counts=None, tokens=1,
             q_heads=8, scale=0.1, accumulate=0)
    v.update(kw)
    return _lib.lib().dq_kv_attend(C.byref(c) if c else None, C.byref(_lib.DqKvAttend(**v)), P(ws), ws_bytes, None)


def evict(c, keep=64, recent=8, sink=2, ws=256, ws_bytes=1 << 40):
    return _lib.lib().dq_kv_evict(C.byref(c) if c else None, keep, recent, sink, P(ws), ws_bytes, None)


def test_sizes():
    L = _lib.lib()
    assert [L.dq_kv_unit_bytes(d) for d in (64, 128, 96, 0, -64, 256)] == [1152, 2176, 0, 0, 0, 0]
    assert unit_bytes(64) == 1152 and unit_bytes(128) == 2176
    c = cache()
    base = L.dq_kv_attend_workspace_bytes(C.byref(c), 1, 8, 0)
    assert base > 0 and base % 256 == 0
    assert L.dq_kv_attend_workspace_bytes(C.byref(c), 1, 8, 1) == base + 256 + 8 * 2 * 64 * 4 * 4  # 2 x 8 log-sums, 4 scores a slot
    assert L.dq_kv_attend_workspace_bytes(C.byref(c), 4, 8, 0) > base        # 16 rows per KV head
    assert L.dq_kv_attend_workspace_bytes(C.byref(c), 1, 7, 0) == 0
    assert L.dq_kv_attend_workspace_bytes(C.byref(cache(head_dim=96)), 1, 8, 0) == 0
    assert L.dq_kv_attend_workspace_bytes(None, 1, 8, 0) == 0
    # two lists of at most min(keep, capacity - keep) entries per sequence and head, and a count
    assert L.dq_kv_evict_workspace_bytes(C.byref(c), 200) == 2 * 2 * 2 * 56 * 4 + (-2 * 2 * 2 * 56 * 4) % 256 + 256
    assert L.dq_kv_evict_workspace_bytes(C.byref(c), 256) == 0
    assert L.dq_kv_evict_workspace_bytes(C.byref(c), 0) == 0


@pytest.mark.parametrize("call", [append, attend, evict], ids=["append", "attend", "evict"])
def test_every_call_checks_the_cache(call):
    inv, shape, align, unsup = (_lib.DQ_ERR_INVALID_ARGUMENT, _lib.DQ_ERR_SHAPE, _lib.DQ_ERR_ALIGNMENT,
                                _lib.DQ_ERR_UNSUPPORTED)
    assert call(None) == inv
    for name in ("units", "mass", "pos", "lengths", "evicted", "page_table", "arrivals"):
        assert call(cache(**{name: None})) == inv, name
        assert call(cache(**{name: 257})) == align, name
    assert call(cache(units=260)) == align
    for bad in (dict(page_size=24), dict(page_size=0), dict(page_size=-16), dict(kv_heads=0), dict(n_seqs=-1),
                dict(n_pages=-1), dict(max_pages=-1)):
        assert call(cache(**bad)) == shape, bad
    for bad in (dict(head_dim=96), dict(head_dim=0), dict(n_seqs=1025), dict(max_pages=1 << 25), dict(kv_heads=1 << 17)):
        assert call(cache(**bad)) == unsup, bad
    assert call(cache(n_seqs=0, lengths=None, evicted=None, arrivals=None)) == _lib.DQ_OK


def test_append_arguments():
    c = cache()
    assert append(c, tokens=-1) == _lib.DQ_ERR_SHAPE
    assert append(c, tokens=0, k=None) == _lib.DQ_OK
    assert append(c, k=None) == _lib.DQ_ERR_INVALID_ARGUMENT
    assert append(c, v=None) == _lib.DQ_ERR_INVALID_ARGUMENT
    assert append(c, kv=256) == _lib.DQ_ERR_INVALID_ARGUMENT  # one of the two value outputs
    assert append(c, k=258) == _lib.DQ_ERR_ALIGNMENT
    assert append(c, counts=258) == _lib.DQ_ERR_ALIGNMENT
    assert append(c, ks=(1024, 256, 132)) == _lib.DQ_ERR_ALIGNMENT
    assert append(c, vs=(-1024, 256, 128)) == _lib.DQ_ERR_ALIGNMENT


def test_attend_arguments():
    c = cache()
    assert attend(c, q_heads=7) == _lib.DQ_ERR_SHAPE
    assert attend(c, q_heads=0) == _lib.DQ_ERR_SHAPE
    assert attend(c, tokens=-1) == _lib.DQ_ERR_SHAPE
    assert attend(c, tokens=1 << 27) == _lib.DQ_ERR_UNSUPPORTED
    assert attend(c, tokens=0, q=None) == _lib.DQ_OK
    assert attend(c, q=None) == _lib.DQ_ERR_INVALID_ARGUMENT
    assert attend(c, out=None) == _lib.DQ_ERR_INVALID_ARGUMENT
    assert attend(c, scale=float("nan")) == _lib.DQ_ERR_INVALID_ARGUMENT
    assert attend(c, scale=float("-inf")) == _lib.DQ_ERR_INVALID_ARGUMENT
    assert attend(c, q_stride=S3(1024, 1024, 100)) == _lib.DQ_ERR_ALIGNMENT
    assert attend(c, out=264) == _lib.DQ_ERR_ALIGNMENT
    assert attend(c, lse=258) == _lib.DQ_ERR_ALIGNMENT
    assert attend(c, ws=None) == _lib.DQ_ERR_WORKSPACE
    assert attend(c, ws_bytes=1024) == _lib.DQ_ERR_WORKSPACE
    assert attend(c, ws=260) == _lib.DQ_ERR_ALIGNMENT
    assert _lib.lib().dq_kv_attend(C.byref(c), None, P(256), 1 << 40, None) == _lib.DQ_ERR_INVALID_ARGUMENT


def test_evict_arguments():
    c = cache()
    for keep, recent, sink in ((0, 0, 0), (-5, 0, 0), (64, 65, 0), (64, 60, 5), (64, -1, 0), (64, 0, -1),
                               (64, 2 ** 31 - 1, 2 ** 31 - 1)):
        assert evict(c, keep, recent, sink) == _lib.DQ_ERR_INVALID_ARGUMENT
    assert evict(c, ws=None) == _lib.DQ_ERR_WORKSPACE
    assert evict(c, ws_bytes=8) == _lib.DQ_ERR_WORKSPACE
    assert evict(c, ws=258) == _lib.DQ_ERR_ALIGNMENT
    assert evict(c, keep=256, ws=None, ws_bytes=0) == _lib.DQ_OK  # no sequence can hold more


def test_python_refusals_without_a_gpu():
    for a, kw in (((2, 4, 2, 96), {}), ((2, 4, 2, 128, 24), {}), ((0, 4, 2), {}), ((2, 0, 2), {}), ((2, 4, 0), {}),
                  ((2, 4, 2), dict(max_pages=0)), ((2, 4, 2), dict(device="cpu"))):
        with pytest.raises(RuntimeError):
            Int4KVCache(*a, **kw)
