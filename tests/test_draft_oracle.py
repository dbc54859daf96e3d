"""The restatement of trees, sampling and acceptance against cases worked out by hand, and what the entry points refuse before any
kernel runs.  No GPU."""
import ctypes
import math

import numpy as np
import pytest

from gomlx_amd import _lib
from oracle import draft_oracle as ref


def test_trees_by_hand():
    sets = ref.ancestors([-1, 0, 0, 1, 9, 2])
    assert sets == [{0}, {0, 1}, {0, 2}, {0, 1, 3}, {4}, {0, 2, 5}]
    assert ref.masks(sets, 1)[:, 0].tolist() == [1, 3, 5, 11, 16, 37]
    assert ref.masks([{31}, {32}, {0, 33}], 2).tolist() == [[-2 ** 31, 0], [0, 1], [1, 2]]
    see = ref.seen(sets, 8, 0)
    assert see[3].tolist() == [True, True, True, True, False, True, False, False]
    assert ref.seen(sets, 8, 3)[3].tolist() == [False, False, True, True, False, True, False, False]
    assert ref.seen(sets, 8, 2)[3].tolist() == [False, False, False, True, False, True, False, False]
    assert ref.seen([set()], 1, 0).tolist() == [[False]]


def test_sampling_by_hand():
    x = np.log(np.array([1.0, 4.0, 2.0, 2.0, 1.0], np.float64))
    pick = lambda u, **how: ref.sample(x, u, **how)[0]  # noqa: E731
    assert [pick(u) for u in (0.0, 0.05, 0.11, 0.49, 0.51, 0.69, 0.71, 0.95)] == [0, 0, 1, 1, 2, 2, 3, 4]
    assert [pick(u, top_k=2) for u in (0.0, 0.66, 0.67, 0.99)] == [1, 1, 2, 2]       # of two equal ones the lower
    assert [pick(u, top_k=1) for u in (0.0, 0.99)] == [1, 1]
    assert [pick(u, top_p=0.4) for u in (0.0, 0.99)] == [1, 1]
    assert [pick(u, top_p=0.41) for u in (0.0, 0.99)] == [1, 2]
    assert [pick(u, top_k=2, top_p=0.66) for u in (0.0, 0.99)] == [1, 1]          # of the first two: 2/3 and 1/3
    assert [pick(u, min_p=0.49) for u in (0.0, 0.99)] == [1, 3]
    assert pick(0.9, temperature=0.0) == 1
    assert ref.sample(np.array([-np.inf, np.nan]), 0.5)[:2] == (-1, 0.0)
    assert ref.sample(np.array([0.0, np.inf, np.inf]), 0.7)[:2] == (2, 0.5)
    assert ref.sample(x, 0.2)[1] == pytest.approx(0.4)


def test_paths_by_hand():
    parents, tokens = [-1, 0, 0, 1, 1, 3], [7, 5, 6, 5, 5, 9]
    assert ref.walk(parents, tokens, [5, 5, 0, 9, 0, 1]) == [0, 1, 3, 5]
    assert ref.walk(parents, tokens, [6, 5, 0, 9, 0, 1]) == [0, 2]
    assert ref.walk(parents, tokens, [-1, 5, 0, 9, 0, 1]) == [0]
    assert ref.walk([], [], []) == []


def _error(rc):
    return rc, _lib.lib().gq_last_error().decode()


class Buffers:
    """Host memory in the place of device memory: what is refused here is refused before anything looks at it."""

    def __init__(self):
        self.memory = (ctypes.c_int32 * 4096)()
        self.at = ctypes.addressof(self.memory) + (-ctypes.addressof(self.memory)) % 16

    def __call__(self, ints=0):
        return self.at + 4 * ints


def test_draft_tree_refusals():
    L, p = _lib.lib(), Buffers()

    def call(parents=None, first=None, starts=None, seqs=2, rows=8, max_new=4, tree=None, words=1, positions=None):
        d = p()
        return _error(L.gq_draft_tree(parents or d, first or d, starts or d, seqs, rows, max_new, tree or d, words, positions or d, None))

    assert call(seqs=-1)[0] == call(rows=-1)[0] == call(max_new=-1)[0] == _lib.ERR_INVALID
    assert call(rows=2000, max_new=1025, words=40)[0] == _lib.ERR_NOT_IMPLEMENTED
    rc, text = call(rows=100, max_new=33, words=1)
    assert rc == _lib.ERR_INVALID and "no bits for 33" in text
    assert call(words=0)[0] == _lib.ERR_INVALID
    assert call(parents=p() + 2)[0] == _lib.ERR_INVALID
    assert _error(L.gq_draft_tree(p(), p(), None, 2, 3, 1, p(), 1, p(), None))[0] == _lib.ERR_INVALID  # a row a sequence
    assert _error(L.gq_draft_tree(None, p(), p(), 2, 3, 2, p(), 1, p(), None))[0] == _lib.ERR_INVALID
    assert _error(L.gq_draft_tree(None, None, p(), 0, 0, 4, None, 1, None, None))[0] == _lib.OK  # nothing to do


def _kv(p, **how):
    d = dict(dCache=p(), pages=2, kv_heads=2, head_dim=64, page_tokens=32, max_pages=2, dPageTable=p(), table_stride=2, dLengths=p(100), dStarts=p(200), seqs=2, rows=8, max_new=4)
    d.update(how)
    return _lib.KvCacheDesc(*(d[n] for n, _ in _lib.KvCacheDesc._fields_))


def test_tree_attention_refusals():
    L, p = _lib.lib(), Buffers()

    def call(heads=4, words=1, window=0, dtype=_lib.F32, tree=True, out=True, q=True, **kv):
        d, r = _kv(p, **kv), _lib.HeadRowsDesc(p() if q else None, 256, 64)
        return _error(L.gq_kv_tree_attention(ctypes.byref(d), dtype, ctypes.byref(r), heads, 1.0, window, p() if tree else None, words, p() if out else None, None))

    for bad in (dict(heads=3), dict(heads=0), dict(window=-1), dict(words=0), dict(words=1, max_new=33, rows=40), dict(tree=False), dict(out=False), dict(q=False), dict(page_tokens=33),
                dict(dLengths=None), dict(table_stride=1), dict(rows=2 ** 31 - 1, max_new=4, heads=4), dict(seqs=60000, kv_heads=4, max_pages=60000, table_stride=60000)):
        assert call(**bad)[0] == _lib.ERR_INVALID, bad
    assert call(dtype=7)[0] == call(head_dim=96)[0] == _lib.ERR_NOT_IMPLEMENTED
    assert call(seqs=0, rows=0)[0] == _lib.OK


def test_sample_refusals():
    L, p = _lib.lib(), Buffers()

    def call(dtype=_lib.F32, logits=True, rows=2, vocab=10, stride=10, u=True, how=True, tokens=True, **fields):
        d = _lib.SamplingDesc(1.0, 1.0, 0.0, 0, **fields)
        return _error(L.gq_sample(dtype, (p() if logits is True else logits), rows, vocab, stride, p() if u else None, ctypes.byref(d) if how else None, p() if tokens else None, None, None))

    for bad in (dict(rows=-1), dict(vocab=0), dict(stride=-1), dict(u=False), dict(how=False), dict(tokens=False), dict(logits=None), dict(logits=p() + 2), dict(dTopP=p() + 1)):
        assert call(**bad)[0] == _lib.ERR_INVALID, bad
    assert call(dtype=5)[0] == _lib.ERR_NOT_IMPLEMENTED
    assert call(rows=0)[0] == _lib.OK


@pytest.mark.parametrize("vocab", [2 ** 21 - 6, 2 ** 21, 2 ** 31, 2 ** 42, 2 ** 43 - 2 ** 11, 2 ** 43, 2 ** 62, 2 ** 63 - 1])
def test_sample_refuses_vocabularies_that_32_bits_do_not_count(vocab):
    L, p = _lib.lib(), Buffers()
    d = _lib.SamplingDesc(1.0, 1.0, 0.0, 0)
    rc, text = _error(L.gq_sample(_lib.F32, p(), 1, vocab, vocab, p(), ctypes.byref(d), p(), None, None))
    assert rc == _lib.ERR_INVALID and f"{vocab} tokens: at most {2 ** 21 - 7}" in text


def test_top_k_is_a_whole_number():
    from gomlx_amd import nn
    for k in (0, 1, 50, 50.0, np.int64(7), np.float32(7), 2 ** 70):
        nn._sampling_number("top_k", k, 0, math.inf)
    for k in (0.5, 2.9, np.float32(1.5), -1, -0.5, math.inf, math.nan):
        with pytest.raises(ValueError, match="top_k"):
            nn._sampling_number("top_k", k, 0, math.inf)
    nn._sampling_number("temperature", 0.5, 0.0, math.inf)
    nn._sampling_number("temperature", math.inf, 0.0, math.inf)
    with pytest.raises(ValueError, match="top_p"):
        nn._sampling_number("top_p", 1.5, 0.0, 1.0)


def test_accept_refusals():
    L, p = _lib.lib(), Buffers()

    def call(parents=300, tokens=400, sampled=500, path=600, columns=4, token=700, lengths=800, **kv):
        d = _kv(p, **kv)
        a = [None if i is None else p(i) for i in (parents, tokens, sampled, path, token, lengths)]
        return _error(L.gq_kv_accept(ctypes.byref(d), a[0], a[1], a[2], None, a[3], columns, a[4], a[5], None))

    for bad in (dict(columns=3), dict(parents=None), dict(sampled=None), dict(path=None), dict(token=None), dict(lengths=None)):
        assert call(**bad)[0] == _lib.ERR_INVALID, bad
    for bad in (dict(lengths=100), dict(lengths=101), dict(token=507), dict(path=293), dict(path=199), dict(token=1)):
        rc, text = call(**bad)
        assert rc == _lib.ERR_INVALID and "overlaps" in text, bad
    assert call(rows=2000, max_new=1025, columns=1025)[0] == _lib.ERR_NOT_IMPLEMENTED
    assert call(seqs=0, rows=0)[0] == _lib.OK
