"""The 4-bit cache without a GPU: the oracle's byte addresses and quantisation, and the entry points' checks of their arguments."""
import ctypes

import numpy as np
import pytest

from gomlx_amd import _lib
from oracle import kv_oracle as ref


@pytest.mark.parametrize("dim", (64, 128, 256))
def test_addresses_cover_a_tile_once(dim):
    seen = np.zeros((36 * dim, 2), int)
    for values in (False, True):
        byte, high, scale = ref._addresses(dim, values)
        np.add.at(seen, (byte, high), 1)
        for s in np.unique(scale):
            seen[s] += 1
            seen[s + 1] += 1
        for t in range(32):  # a group has one scale
            assert np.all(scale[t].reshape(-1, 32) == scale[t].reshape(-1, 32)[:, :1])
    assert np.all(seen == 1)


def test_quantised_values_are_half_precision_numbers_and_near():
    rng = np.random.default_rng(0)
    for size in (1e-6, 1e-3, 1.0, 1e4):
        k, v = (np.clip(size * rng.standard_normal((50, 128)), -65000, 65000).astype(np.float32) for _ in range(2))
        for x, y in zip((k, v), ref.quantise(k, v)):
            assert np.array_equal(y, y.astype(np.float16).astype(np.float64))
            top = np.abs(x).reshape(50, 4, 32).max(-1)
            step = top / 8 * (1 + 2.0 ** -8) + 2.0 ** -24
            # half a step, or a whole one for the largest of the sign that has seven steps; a scale off by 2^-9 (or a denormal's rounding) over eight
            assert np.all(np.abs(x - y).reshape(50, 4, 32) <= (step + top * 2.0 ** -8 + 8 * 2.0 ** -24)[..., None])
    k, v = ref.quantise(np.zeros((1, 64), np.float32), np.full((1, 64), 65408.0, np.float32))
    assert np.isnan(k).all() and np.all(v == 0)


def _desc(**change):
    d = dict(dCache=1 << 20, pages=4, kv_heads=2, head_dim=128, page_tokens=64, max_pages=3, dPageTable=1 << 12, table_stride=3, dLengths=1 << 12, dStarts=None, seqs=2,
             rows=2, max_new=1)
    d.update(change)
    return ctypes.byref(_lib.KvCacheDesc(*[d[f] for f, _ in _lib.KvCacheDesc._fields_]))


ROWS = ctypes.byref(_lib.HeadRowsDesc(1 << 12, 256, 128))
OUT = 1 << 16


def _attend(kv, dtype=_lib.F32, rows=ROWS, heads=4, window=0, accounts=None, out=OUT):
    return _lib.lib().gq_kv_attention(kv, dtype, rows, heads, 1.0, window, accounts, out, None)


BAD = [dict(page_tokens=48), dict(page_tokens=0), dict(kv_heads=0), dict(pages=-1), dict(seqs=-1), dict(seqs=70000, rows=70000), dict(rows=3), dict(max_new=0),
       dict(dCache=8), dict(dLengths=None), dict(dPageTable=None), dict(dCache=None), dict(dLengths=2), dict(dStarts=2), dict(table_stride=2), dict(pages=1 << 40),
       dict(max_pages=1 << 30, table_stride=1 << 30), dict(rows=-1, dStarts=1 << 12), dict(rows=1 << 40, dStarts=1 << 12)]


@pytest.mark.parametrize("bad", BAD, ids=[str(b) for b in BAD])
def test_entry_points_refuse_malformed_caches(bad):
    L = _lib.lib()
    assert _attend(_desc(**bad)) == _lib.ERR_INVALID
    assert L.gq_kv_append(_desc(**bad), _lib.F32, ROWS, ROWS, None, None) == _lib.ERR_INVALID
    assert L.gq_kv_read(_desc(**bad), OUT, OUT, None) == _lib.ERR_INVALID
    assert L.gq_last_error()


def test_entry_points_refuse_other_arguments():
    L = _lib.lib()
    assert _attend(None) == _lib.ERR_INVALID
    assert _attend(_desc(head_dim=80)) == _lib.ERR_NOT_IMPLEMENTED
    assert _attend(_desc(), dtype=7) == _lib.ERR_NOT_IMPLEMENTED
    for bad in (dict(heads=3), dict(heads=0), dict(window=-1), dict(rows=None), dict(out=None), dict(out=8), dict(accounts=2),
                dict(rows=ctypes.byref(_lib.HeadRowsDesc(1 << 12, -1, 0))), dict(rows=ctypes.byref(_lib.HeadRowsDesc(2, 1, 0)))):
        assert _attend(_desc(), **bad) == _lib.ERR_INVALID, bad
    assert _attend(_desc(dStarts=1 << 12, rows=1 << 30, max_new=1 << 20)) == _lib.ERR_INVALID  # a grid past 32 bits
    for keep, recent in ((0, 0), (4, 5), (4, -1), (1 << 40, 0)):
        assert L.gq_kv_evict(_desc(), OUT, keep, recent, OUT, OUT, None) == _lib.ERR_INVALID
    assert L.gq_kv_evict(_desc(), None, 4, 0, OUT, OUT, None) == _lib.ERR_INVALID

    def rope(dtype=_lib.F32, rows=ROWS, heads=4, dim=128, n=2, pos=OUT, cos=OUT, rot=128, out_type=_lib.F32, out=OUT, norm=None):
        return L.gq_qk_norm_rope(dtype, rows, heads, rows, 2, dim, n, pos, cos, cos, 10, rot, 0, norm, None, out_type, out, out, None)
    assert rope(dim=96) == rope(dtype=3) == rope(out_type=3) == _lib.ERR_NOT_IMPLEMENTED
    for bad in (dict(rot=12), dict(rot=136), dict(rot=-8), dict(n=-1), dict(heads=-1), dict(pos=None), dict(cos=None), dict(cos=8), dict(out=None), dict(out=4), dict(rows=None),
                dict(n=1 << 30, heads=1 << 10), dict(norm=ctypes.byref(_lib.RmsNormDesc(2, 0.0, 0.0)))):
        assert rope(**bad) == _lib.ERR_INVALID, bad


def test_empty_calls_need_no_device():
    L = _lib.lib()
    none = dict(seqs=0, rows=0)
    assert _attend(_desc(**none)) == _lib.OK
    assert L.gq_kv_append(_desc(**none), _lib.F32, ROWS, ROWS, None, None) == _lib.OK
    assert L.gq_kv_read(_desc(**none), None, None, None) == _lib.OK
    assert L.gq_kv_evict(_desc(**none), None, 4, 0, None, None, None) == _lib.OK


def test_nn_refuses_tensors_off_the_gpu():
    import torch
    from gomlx_amd import nn
    cache = torch.zeros(1, 1, 1, 36 * 64, dtype=torch.uint8)
    n = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        nn.cached_attention(torch.zeros(1, 1, 64), cache, n.view(1, 1), n)
    with pytest.raises(ValueError, match="GPU"):
        nn.qk_norm_rope(torch.zeros(1, 1, 64), torch.zeros(1, 1, 64), n, torch.zeros(1, 32), torch.zeros(1, 32))
    cos, sin = nn.rotary_table(4, 8, 10.0, device="cpu")
    assert np.allclose(sin.numpy(), np.sin(np.arange(4)[:, None] * 10.0 ** (-np.arange(0, 8, 2) / 8)), atol=1e-7)
