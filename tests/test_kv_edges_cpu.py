"""The KV cache's C entry points on a host without a GPU, where sizes are at their edges."""
import ctypes as C

import pytest
import torch

from dyn_quant import _lib
from dyn_quant.attention import Int4Attention
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


def test_attention_layer_refuses_projections_of_other_shapes():
    """Also where the stacked matrix would have the right size: wq and wk exchanged."""
    layer = Int4Attention(256, 4, 2, 64)
    wq, wk, wo = torch.zeros(256, 256), torch.zeros(128, 256), torch.zeros(256, 256)
    for w in ((wk, wq, wk, wo), (wk, wk, wq, wo), (wq, wk, wk[:64], wo), (wq, wk, wk, wo[:128]), (wq[:, :128], wk, wk, wo)):
        with pytest.raises(RuntimeError, match="must be"):
            layer.load_weights(*w)


def test_attend_refuses_scales_whose_products_overflow():
    """1e29 times log2(e), 2^14 and the largest f16 scale is below the largest FP32 number."""
    c = cache()
    assert 1e29 * 1.4427 * 2 ** 14 * 65504 < 3.4e38
    for scale in (1.01e29, -1e30, 3e38):
        assert attend(c, scale=scale) == _lib.DQ_ERR_INVALID_ARGUMENT
    for scale in (1e29, -1e29, 0.0):
        assert attend(c, scale=scale, ws_bytes=8) == _lib.DQ_ERR_WORKSPACE
