"""Decoding with drafted tokens on the GPU against its definition in 64 bits (oracle/draft_oracle.py, oracle/kv_oracle.py)."""
import itertools
import math

import numpy as np
import pytest

from oracle import draft_oracle as ref
from oracle import kv_oracle as kv_ref
from tests.test_kv_attention_gpu import EPS, Case, attention_bound

pytestmark = pytest.mark.gpu


def random_parents(rng, n, bend=2.0):
    return [-1] + [int(i * rng.random() ** bend) for i in range(1, n)]


def ints(torch, v):
    return torch.tensor(np.asarray(v, dtype=np.int32), device="cuda")


def starts_of(news):
    return np.concatenate([[0], np.cumsum(news)])


# ---- trees ------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("news,max_new", [([1], 1), ([8], 8), ([31, 1, 32, 33, 0, 64, 65], 65), ([1024, 3], 1024), ([200, 100], 777)])
def test_tree_masks_and_positions(gpu, news, max_new):
    torch = gpu
    from gomlx_amd import nn
    rng = np.random.default_rng(sum(news))
    parents = [random_parents(rng, n) if n else [] for n in news]
    if news[0] > 100:
        parents[0] = list(range(-1, news[0] - 1))  # a chain
    for p in parents:  # parents that are none: behind their child, the child itself, far out
        for i, bad in zip(range(len(p) - 1, 5, -7), itertools.cycle((10 ** 9, -2 ** 31, None, -5))):
            p[i] = i if bad is None else bad
    first = rng.integers(0, 10000, len(news))
    tree, positions = nn.draft_tree(ints(torch, sum(parents, [])), ints(torch, first), starts=ints(torch, starts_of(news)), max_new=max_new)
    assert tree.shape == (sum(news), -(-max_new // 32))
    sets = [ref.ancestors(p) for p in parents]
    assert np.array_equal(tree.cpu().numpy(), np.concatenate([ref.masks(s, tree.shape[1]) for s in sets]))
    assert positions.tolist() == [int(f) + len(x) - 1 for f, s in zip(first, sets) for x in s]


def test_tree_of_one_row_a_sequence(gpu):
    torch = gpu
    from gomlx_amd import nn
    tree, positions = nn.draft_tree(ints(torch, [-1, 0, 5]), ints(torch, [7, 0, 9]))
    assert tree.tolist() == [[1], [1], [1]] and positions.tolist() == [7, 0, 9]


def test_tree_rows_that_are_left_out(gpu):
    """More rows than max_new in a sequence, rows behind the last sequence, starts that lead out of the call: what no sequence has is left as it is."""
    torch = gpu
    import ctypes
    from gomlx_amd import _lib
    rows, words = 12, 1
    parents, first = ints(torch, [-1, 0, 1, 2, 3, 4, -1, 0, 0, 1, 0, 0]), ints(torch, [0, 50])
    for starts, written in (([0, 6, 9], {0, 1, 2, 3, 6, 7, 8}), ([0, 6, 99], {0, 1, 2, 3, 6, 7, 8, 9}), ([-5, 2, 1], {0, 1})):
        tree, positions = torch.full((rows, words), 77, dtype=torch.int32, device="cuda"), torch.full((rows,), 77, dtype=torch.int32, device="cuda")
        s = ints(torch, starts)
        _lib.check(_lib.lib().gq_draft_tree(parents.data_ptr(), first.data_ptr(), s.data_ptr(), 2, rows, 4, tree.data_ptr(), words, positions.data_ptr(), ctypes.c_void_p(0)))
        torch.cuda.synchronize()
        assert {i for i in range(rows) if tree[i, 0] != 77} == written
        assert {i for i in range(rows) if positions[i] != 77} == written


# ---- attention ----------------------------------------------------------------------------------------------------------


def check_attention(c, news, heads, sets, dtype="f32", window=0, q=None, scale=None, table=None, absent=None, words=None, call=None):
    """tree_attention of a Case's last rows against 64 bits, within the bound of attention over the same operands."""
    torch, group, rows = c.torch, heads // c.kv_heads, sum(news)
    if q is None:
        q = torch.from_numpy(c.rng.standard_normal((rows, heads, c.dim)).astype(np.float32)).cuda()
    q = q.to({"f32": torch.float32, "bf16": torch.bfloat16}[dtype])
    words = -(-max(news) // 32) if words is None else words
    tree = torch.from_numpy(np.concatenate([ref.masks(s, words) for s in sets if len(s)])).cuda()
    single = all(n == 1 for n in news)
    starts = None if single else c.ints(starts_of(news))
    args = dict(starts=starts, max_new=1 if single else max(news), window=window, scale=scale)
    out = (call or c.nn.tree_attention)(q, c.cache, c.d_table if table is None else table, c.ints(c.lengths), tree, **args)
    assert out.dtype == q.dtype and out.shape == q.shape and out.is_contiguous()
    got_all, q = out.double().cpu().numpy(), q.double().cpu().numpy()
    host, at = c.host(), 0
    scale = c.dim ** -0.5 if scale is None else scale
    for b, n in enumerate(news):
        see = ref.seen(sets[b], c.lengths[b], window)
        if absent is not None:
            see[:, absent[b]] = False
        for h in range(c.kv_heads):
            keys, values = kv_ref.decode(host, np.maximum(c.table[b], 0), c.lengths[b], h)
            qb = q[at:at + n, h * group:(h + 1) * group]
            want, p, s = ref.attention(qb, keys, values, scale, see)
            got = got_all[at:at + n, h * group:(h + 1) * group]
            assert np.all(got[~see.any(-1)] == 0)
            bound, _ = attention_bound(qb, keys, values, abs(scale), p, s, see, dtype)  # (an error of a score is scale times one of its product, of either sign: |ds| <= |scale| ...)
            bad = np.isnan(want).any(-1)
            assert np.isnan(got[bad]).all()
            off = np.abs(got - want) - bound - np.abs(want) * (2.0 ** -8 if dtype == "bf16" else 2 * EPS)
            assert np.all(off[~bad] <= 0), f"sequence {b}, head {h}: {np.max(off[~bad])}"
        at += n
    return out


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("dim", (64, 128, 256))
@pytest.mark.parametrize("group,news,lengths", [
    (1, [1, 1], [1, 90]),                    # trees of a root
    (4, [2, 4], [2, 33]),                    # 16 rows and fewer; no context at all
    (8, [3, 4, 2], [100, 64, 40]),           # 32
    (3, [13, 20, 7], [13 + 31, 20 + 32, 7 + 160]),  # 64; trees that begin at, in front of and behind a tile's end
    (4, [33, 16, 40], [300, 500, 41]),       # several blocks of rows, two words of bits
    (7, [5, 0, 11], [200, 3, 11]),           # a sequence without rows
])
def test_attention_over_trees(gpu, dim, dtype, group, news, lengths):
    torch = gpu
    c = Case(torch, lengths, kv_heads=2, dim=dim, page=32 if dim == 64 else 96, seed=dim + group).fill()
    sets = [ref.ancestors(random_parents(c.rng, n)) if n else [] for n in news]
    check_attention(c, news, 2 * group, sets, dtype)


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("window", (1, 2, 7, 40, 64, 10 ** 9))
def test_attention_in_a_window(gpu, dtype, window):
    torch = gpu
    c = Case(torch, [170, 37, 70], page=32, seed=window % 97).fill()
    news = [37, 37, 5]
    sets = [ref.ancestors(random_parents(c.rng, n, 0.5)) for n in news]  # (deep ones: a window of 7 ends inside the tree)
    assert max(len(x) for s in sets for x in s) > 7
    check_attention(c, news, 8, sets, dtype, window=window)


@pytest.mark.parametrize("window", (0, 5))
def test_attention_with_any_masks(gpu, window):
    """Masks that are no tree's: later rows, not the row itself, nothing at all; bits behind the last row count for nothing."""
    torch = gpu
    c = Case(torch, [60, 35, 9], dim=64, page=32, seed=3).fill()
    news = [35, 35, 9]
    sets = [[set(np.nonzero(c.rng.random(n) < 0.3)[0].tolist()) for _ in range(n)] for n in news]
    sets[1][4] = sets[1][34] = sets[0][7] = set()
    for s in sets[2]:
        s.update((9, 20, 31, 33, 63))
    check_attention(c, news, 8, sets, window=window)


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("dim,lengths,news,group", [(128, [9000], [24], 4), (64, [5000, 7], [40, 3], 2), (256, [3000, 1234, 2000], [9, 8, 7], 4), (128, [4000] * 3, [4] * 3, 4)])
def test_attention_over_long_caches_is_joined_from_pieces(gpu, dim, lengths, news, group, dtype):
    torch = gpu
    c = Case(torch, lengths, kv_heads=2, dim=dim, page=64, seed=dim).fill()
    sets = [ref.ancestors(random_parents(c.rng, n)) for n in news]
    check_attention(c, news, 2 * group, sets, dtype)


def test_attention_over_more_than_64_sequences(gpu):
    torch = gpu
    rng = np.random.default_rng(1)
    news = [int(n) for n in rng.integers(0, 6, 150)]
    news[70] = 40
    lengths = [n + int(x) for n, x in zip(news, rng.integers(0, 80, 150))]
    c = Case(torch, lengths, kv_heads=1, dim=64, page=32, seed=2).fill()
    check_attention(c, news, 4, [ref.ancestors(random_parents(rng, n)) if n else [] for n in news], "bf16")


def test_attention_of_one_large_tree_beside_small_ones(gpu):
    torch = gpu
    rng = np.random.default_rng(3)
    news = [int(n) for n in rng.integers(0, 3, 90)]
    news[66] = 300
    lengths = [n + int(x) for n, x in zip(news, rng.integers(0, 300, 90))]
    for dim in (64, 256):
        c = Case(torch, lengths, kv_heads=2, dim=dim, page=32, seed=2).fill()
        check_attention(c, news, 6, [ref.ancestors(random_parents(rng, n)) if n else [] for n in news], "bf16")


def test_a_chain_is_attention_of_new_tokens(gpu):
    torch = gpu
    c = Case(torch, [500, 90], seed=5).fill()
    news = [20, 13]
    q = torch.randn(33, 8, 128, device="cuda")
    chain = check_attention(c, news, 8, [ref.ancestors(range(-1, n - 1)) for n in news], q=q)
    _, plain = c.attend(news, 8, q=q)
    assert np.allclose(chain.double().cpu().numpy(), plain, rtol=0, atol=1e-5)  # (values of size 1: each within 1e-6 of 64 bits by the bound above)


def test_tokens_that_are_numbers_to_no_one_who_does_not_see_them(gpu):
    """A NaN among drafted tokens: rows that see it are NaN, the others do not notice; absent pages, a table with room to spare."""
    torch = gpu
    c = Case(torch, [100, 70], page=32, wide_table=3, seed=6)
    c.k[0][95, 1, 3] = np.nan
    c.v[1][10, 0, 5] = np.inf
    c.fill()
    news = [10, 6]
    sets = [ref.ancestors(random_parents(c.rng, n)) for n in news]
    sets[0][0], sets[0][9] = {0}, {9}
    sets[0][5] = {0, 5}
    out = check_attention(c, news, 8, sets)
    assert torch.isnan(out[5, 4:]).all() and not torch.isnan(out[0]).any() and not torch.isnan(out[9]).any()
    assert torch.isnan(out[10:, :4]).all() and not torch.isnan(out[10:, 4:]).any()
    # a page that is none of the cache's: its tokens are not there
    c = Case(torch, [100, 70], page=32, seed=7).fill()
    table = c.table.copy()
    table[0, 1], table[1, 2] = -1, c.pages
    sets = [ref.ancestors(random_parents(c.rng, n)) for n in news]
    check_attention(c, news, 8, sets, table=torch.from_numpy(table).cuda(), absent=[slice(32, 64), slice(64, 96)])
    # a table too short for the sequence: what lies behind it is not there, the others keep their places
    check_attention(c, news, 8, sets, table=c.d_table[:, :2].contiguous(), absent=[slice(64, 200), slice(64, 200)])


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
def test_strided_and_unaligned_queries(gpu, dtype):
    torch = gpu
    c = Case(torch, [130], dim=64, seed=8).fill()
    wide = torch.randn(9, 8 * 64 + 7, device="cuda").to(torch.float32 if dtype == "f32" else torch.bfloat16)
    q = wide.as_strided((9, 8, 64), (519, 64, 1), 3)
    check_attention(c, [9], 8, [ref.ancestors(random_parents(c.rng, 9))], dtype, q=q)


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
def test_scores_that_grow_along_the_sequence(gpu, dtype):
    """The rows' references move again and again; scales of either sign."""
    torch = gpu
    c = Case(torch, [400], dim=128, page=64, seed=9)
    c.k[0] *= np.linspace(0.01, 3.0, 400, dtype=np.float32)[:, None, None] ** 2
    c.fill()
    for scale in (0.7, -0.7, 0.0):
        check_attention(c, [20], 8, [ref.ancestors(random_parents(c.rng, 20))], dtype, scale=scale)


def test_attention_replays_from_a_graph_and_on_two_streams(gpu):
    """Recorded with workspaces in use; replays follow lengths and masks on the device, with eager calls of the same stream and another in between."""
    torch = gpu
    from gomlx_amd import nn
    c = Case(torch, [3000, 2500], seed=10).fill()
    news = [16, 16]
    starts, lengths = c.ints(starts_of(news)), c.ints([2000, 1900])
    sets = [[ref.ancestors(random_parents(c.rng, 16)) for _ in news] for _ in range(3)]
    masks = [torch.from_numpy(np.concatenate([ref.masks(s, 1) for s in ss])).cuda() for ss in sets]
    q, tree = torch.randn(32, 16, 128, device="cuda"), masks[0].clone()
    call = lambda: nn.tree_attention(q, c.cache, c.d_table, lengths, tree, starts=starts, max_new=16)  # noqa: E731
    s, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s):
        call()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = call()
    for i in range(6):
        lengths.copy_(c.ints([2000 + 150 * i, 1900 + 100 * i]))
        tree.copy_(masks[i % 3])
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graph.replay()
        with torch.cuda.stream(other):
            elsewhere = call()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            eager = call()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(elsewhere, eager)


def test_attention_refuses(gpu):
    torch = gpu
    from gomlx_amd import _lib, nn
    c = Case(torch, [40, 50]).fill()
    q, tree, starts = torch.randn(7, 4, 128, device="cuda"), torch.ones(7, 1, dtype=torch.int32, device="cuda"), c.ints([0, 3, 7])
    good = dict(q=q, cache=c.cache, page_table=c.d_table, lengths=c.ints([40, 50]), tree=tree, starts=starts, max_new=4)
    nn.tree_attention(**good)
    for bad in (dict(tree=tree.long()), dict(tree=tree[:6]), dict(tree=tree[:, :0]), dict(tree=tree.cpu()), dict(q=q.cpu()), dict(q=q[:, :3]), dict(window=-1), dict(max_new=0), dict(starts=None),
                dict(q=q[..., :64].contiguous()), dict(lengths=c.ints([40]))):
        with pytest.raises(ValueError):
            nn.tree_attention(**{**good, **bad})
    with pytest.raises(_lib.NotImplementedByBackend):
        nn.tree_attention(**{**good, "q": q.half()})


# ---- sampling -----------------------------------------------------------------------------------------------------------


def check_samples(torch, x, u, **how):
    """Tokens equal those of 64 bits, but where a border lies as near to u (or to top-p) as sums may be off: weights are good to 1e-11 and, as whole numbers of 2^-42 of
    the largest, to 2^-43 each, of a sum that is one such largest weight at least; 2 (1e-11 + V 2^-43) for a share of V tokens (a sum over another).  Such a row is met once in thousands,
    where it is the next token in index.  Shares to float32, and with the sum's error."""
    from gomlx_amd import nn
    settings = {k: (torch.from_numpy(v).cuda() if isinstance(v, np.ndarray) else v) for k, v in how.items()}
    u_d = torch.from_numpy(np.asarray(u, np.float32)).cuda()
    tokens, shares = nn.sample(x, u_d, probabilities=True, **settings)
    assert tokens.dtype == torch.int32 and shares.dtype == torch.float32
    assert torch.equal(tokens, nn.sample(x, u_d, **settings))
    host, tokens, shares = x.float().cpu().numpy(), tokens.cpu().numpy(), shares.cpu().numpy()
    near = 2 * (1e-11 + host.shape[1] * 2.0 ** -43)
    for r in range(len(host)):
        row = {k: (v[r].item() if isinstance(v, np.ndarray) else v) for k, v in how.items()}
        token, share, edge = ref.sample(host[r], float(np.float32(u[r])), **row)
        assert tokens[r] == token or edge <= near, f"row {r}: {tokens[r]} for {token}, {edge} from a border"
        if tokens[r] == token and edge > near:
            assert abs(shares[r] - share) <= (2 * EPS + near) * share
    return tokens


def logits(rng, rows, vocab, sure=True):
    x = 1.5 * rng.standard_normal((rows, vocab))
    if sure:
        for r in range(rows):
            n = min(vocab, 200)
            at = rng.choice(vocab, n, replace=False)
            x[r, at] = rng.uniform(10, 22) - 1.5 * np.log(np.arange(1, n + 1)) + 0.5 * rng.standard_normal(n)
    return x.astype(np.float32)


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7), dict(top_k=1), dict(top_k=20), dict(top_k=300, temperature=1.3), dict(top_p=0.9), dict(top_p=0.3), dict(top_p=0.0),
            dict(min_p=0.1), dict(min_p=1.0), dict(min_p=1e-6), dict(top_k=50, top_p=0.95, temperature=0.8), dict(top_k=40, top_p=0.9, min_p=0.05), dict(top_p=0.999, min_p=0.02, temperature=0.6)]


@pytest.mark.parametrize("how", SETTINGS, ids=lambda h: "-".join(f"{k}{v}" for k, v in h.items()) or "plain")
@pytest.mark.parametrize("vocab,dtype", [(1, "f32"), (7, "bf16"), (2048, "f32"), (2051, "bf16"), (32003, "f32"), (50257, "bf16")])
def test_samples(gpu, vocab, dtype, how):
    torch = gpu
    rng = np.random.default_rng(vocab)
    rows = 9 if vocab > 10000 else 21
    x = torch.from_numpy(logits(rng, rows, vocab)).cuda().to(torch.float32 if dtype == "f32" else torch.bfloat16)
    u = rng.random(rows)
    u[0], u[1] = 0.0, 1.0 - 2.0 ** -24
    check_samples(torch, x, u, **how)


@pytest.mark.parametrize("how", SETTINGS + [dict(top_k=300, top_p=0.9), dict(top_k=3000, top_p=0.7, min_p=0.05), dict(top_k=3000, top_p=0.9, min_p=0.3), dict(top_k=39999, top_p=0.9),
                                            dict(top_k=20000, top_p=0.001), dict(top_k=20000, min_p=0.01)], ids=lambda h: "-".join(f"{k}{v}" for k, v in h.items()) or "plain")
def test_samples_of_flat_distributions(gpu, how):
    """The cut lies below what the first launch leaves of each chunk: the row is gone over again."""
    torch = gpu
    rng = np.random.default_rng(4)
    x = logits(rng, 6, 40001, sure=False)
    x[1] = 0.25 * np.round(4 * x[1])     # a few values, each many times
    x[2] = -1.5                          # one value
    x[3] *= 0.001
    x[4] *= 40.0
    check_samples(torch, torch.from_numpy(x).cuda(), rng.random(6), **how)
    check_samples(torch, torch.from_numpy(x).cuda().bfloat16(), rng.random(6), **how)


@pytest.mark.parametrize("how", [dict(), dict(top_k=3), dict(top_k=5000), dict(top_p=0.6), dict(min_p=0.3), dict(top_k=2500, top_p=0.9), dict(temperature=0.0), dict(temperature=1e-30),
                                 dict(temperature=1e30), dict(temperature=math.inf, top_p=0.5)], ids=str)
def test_samples_of_rows_with_holes(gpu, how):
    """Minus infinity, NaN and infinity; both zeros, which are equal; rows with one number and with none."""
    torch = gpu
    rng = np.random.default_rng(5)
    x = logits(rng, 8, 5000, sure=False)
    x[0, rng.random(5000) < 0.7] = -np.inf
    x[1, rng.random(5000) < 0.5] = np.nan
    x[2] = -np.inf
    x[2, 4321] = -3e38
    x[3] = np.where(rng.random(5000) < 0.5, -np.inf, np.nan)
    x[4, [17, 4000]] = np.inf
    x[5] = np.where(rng.random(5000) < 0.5, 0.0, -0.0)
    x[6] = np.where(rng.random(5000) < 0.01, 3e38, -3e38)
    x[7, :4999] = -np.inf
    tokens = check_samples(torch, torch.from_numpy(x).cuda(), rng.random(8), **how)
    assert tokens[3] == -1 and tokens[2] == 4321 and tokens[7] == 4999 and tokens[4] in (17, 4000)


def kernel_us(call, times=15):
    """The least time that the kernels of a call have taken."""
    import ctypes
    from gomlx_amd import _lib
    n, us, out = ctypes.c_int(), ctypes.c_double(), []
    for _ in range(times):
        _lib.check(_lib.lib().gq_profile_begin())
        call()
        _lib.check(_lib.lib().gq_profile_end(ctypes.byref(n), ctypes.byref(us)))
        out.append(us.value)
    return min(out)


def masked(rng, x, allowed, value):
    """All but `allowed` tokens of every row at one value."""
    out = np.full_like(x, value)
    for r in range(len(x)):
        keep = np.concatenate([np.argsort(-x[r])[:allowed // 2], rng.choice(x.shape[1], allowed - allowed // 2, replace=False)])
        out[r, keep] = x[r, keep]
    return out


@pytest.mark.parametrize("how", [dict(top_k=50, top_p=0.9, temperature=0.8), dict(top_k=50), dict(top_k=3), dict(top_p=0.9), dict(top_p=0.9999), dict(min_p=0.05), dict(min_p=1e-9), dict(top_k=200, top_p=0.95),
                                 dict(top_k=3000, min_p=0.01), dict(top_k=40, temperature=30.0), dict(top_p=0.5, temperature=1e9)], ids=str)
@pytest.mark.parametrize("dtype", ("f32", "bf16"))
def test_samples_of_rows_with_many_equal_logits(gpu, how, dtype):
    torch = gpu
    rng = np.random.default_rng(14)
    vocab = 20003
    x = logits(rng, 10, vocab)
    x[0] = masked(rng, x[:1], 300, -1e9)[0]
    x[1] = masked(rng, x[1:2], 12, -1e9)[0]
    x[2] = masked(rng, x[2:3], 2000, -30.0)[0]
    x[3, 5000:] = 0.0                         # padding, of chunks that have nothing else
    x[4, 12000:16000] = 9.0                   # among the likely ones
    x[5] = np.where(rng.random(vocab) < 0.001, 4.0, np.where(rng.random(vocab) < 0.1, 3.0, -2.0))
    x[6, rng.random(vocab) < 0.1] = np.inf
    x[7] = -1e9
    x[8] = -20.0
    x[8, (np.arange(vocab) // 4) % 64 < 10] = 1.0 + np.arange(vocab)[(np.arange(vocab) // 4) % 64 < 10] * 1e-4  # all large ones of a chunk in ten lanes
    x[9] = masked(rng, x[9:], 400, -3e38)[0]
    check_samples(torch, torch.from_numpy(x).cuda().to(torch.float32 if dtype == "f32" else torch.bfloat16), rng.random(10), **how)


@pytest.mark.parametrize("how", [dict(top_k=50, top_p=0.9, temperature=0.8), dict(top_k=50), dict(top_p=0.9)], ids=str)
@pytest.mark.parametrize("value", (-1e9, -200.0))
def test_a_mask_by_a_finite_value_takes_no_longer(gpu, how, value):
    """... than one by minus infinity: chunks full of equal logits leave the others' lists alone.  (A row that is gone over alone takes five times as long and more.)"""
    torch = gpu
    from gomlx_amd import nn
    rng = np.random.default_rng(15)
    x = logits(rng, 1, 128256)
    u = torch.rand(1, device="cuda")
    times = []
    for v in (-np.inf, value):
        d = torch.from_numpy(masked(np.random.default_rng(16), x, 300, v)).cuda()
        nn.sample(d, u, **how)
        times.append(kernel_us(lambda: nn.sample(d, u, **how)))  # noqa: B023
    assert times[1] <= 2 * times[0], times
    # padding behind the vocabulary, which ends anywhere in a chunk of 2048
    for rest in (0, 130, 180, 190, 300, 1500):
        x[0, -3000 - rest:] = 0.0
        d = torch.from_numpy(x).cuda()
        padded = kernel_us(lambda: nn.sample(d, u, **how))  # noqa: B023
        x[0, -3000 - rest:] = -np.inf
        e = torch.from_numpy(x).cuda()
        assert padded <= 2 * kernel_us(lambda: nn.sample(e, u, **how)), rest  # noqa: B023


@pytest.mark.parametrize("how", [dict(top_k=50, top_p=0.9, temperature=0.8), dict(top_k=50), dict(top_k=300, top_p=0.99), dict(top_k=50, min_p=0.01), dict(top_k=50, min_p=1e-300),
                                 dict(top_k=50, temperature=0.01), dict(top_k=50, top_p=0.9, temperature=7.0), dict(top_k=40, temperature=1e12)], ids=str)
@pytest.mark.parametrize("dtype", ("f32", "bf16"))
def test_samples_of_rows_with_fewer_tokens_than_top_k(gpu, how, dtype):
    torch = gpu
    rng = np.random.default_rng(17)
    x = np.concatenate([masked(rng, logits(rng, 1, 20003), n, v) for v in (-np.inf, -1e9, -200.0, -20.0, 0.0) for n in (2, 10, 47)])
    x = np.concatenate([x, np.full((2, 20003), -3e38, np.float32)])
    x[-1, 7], x[-2, [5, 19000]] = -2.9e38, 3e38
    check_samples(torch, torch.from_numpy(x).cuda().to(torch.float32 if dtype == "f32" else torch.bfloat16), rng.random(len(x)), **how)


@pytest.mark.parametrize("how", [dict(top_k=50, top_p=0.9, temperature=0.8), dict(top_k=50), dict(top_k=300, top_p=0.9)], ids=str)
@pytest.mark.parametrize("value", (-np.inf, -1e9, -200.0))
def test_a_mask_that_leaves_fewer_tokens_than_top_k_takes_no_longer(gpu, how, value):
    """... than the same under a top-k that they reach: what is masked weighs nothing, so that the row need not be gone over for more."""
    torch = gpu
    from gomlx_amd import nn
    rng = np.random.default_rng(18)
    x, u = torch.from_numpy(masked(rng, logits(rng, 1, 128256), 10, value)).cuda(), torch.rand(1, device="cuda")
    times = []
    for k in (5, how["top_k"]):
        nn.sample(x, u, **{**how, "top_k": k})
        times.append(kernel_us(lambda: nn.sample(x, u, **{**how, "top_k": k})))  # noqa: B023
    # (a top-k of more than 64 has the launches for flat rows behind it, three of which find nothing to do: each some 3 us)
    assert times[1] <= 2 * times[0] + (10 if how["top_k"] > 64 else 0), times


def test_samples_of_more_flat_rows_than_their_launches_take(gpu):
    torch = gpu
    rng = np.random.default_rng(10)
    x = logits(rng, 150, 20000, sure=False)
    x[::7] = np.round(x[::7])
    for how in (dict(top_p=0.8), dict(top_k=3000), dict(min_p=0.01), dict(top_p=0.9, min_p=0.02), dict(top_k=2000, top_p=0.8, min_p=0.01)):
        check_samples(torch, torch.from_numpy(x).cuda(), rng.random(150), **how)


def test_samples_with_settings_of_each_row(gpu):
    torch = gpu
    rng = np.random.default_rng(6)
    rows = 300
    x = torch.from_numpy(logits(rng, rows, 3001)).cuda()
    check_samples(torch, x, rng.random(rows), temperature=rng.choice([0.0, 0.5, 1.0, 2.0], rows).astype(np.float32), top_k=rng.choice([0, 1, 7, 100, 3001, 9999], rows).astype(np.int32),
                  top_p=rng.choice([1.0, 0.5, 0.9], rows).astype(np.float32), min_p=rng.choice([0.0, 0.1], rows).astype(np.float32))
    # out of range and NaN, as the nearest in it and as no bound
    n = 6
    nan = float("nan")
    t, k = np.array([nan, -1, 1, 1, 1, 1], np.float32), np.array([0, 0, -5, 0, 0, 0], np.int32)
    p, m = np.array([1, 1, 1, nan, -1, 2], np.float32), np.array([0, 0, nan, 0, -1, 2], np.float32)
    from gomlx_amd import nn
    u = torch.from_numpy(rng.random(n).astype(np.float32)).cuda()
    d = lambda v: torch.from_numpy(v).cuda()  # noqa: E731
    got = nn.sample(x[:n], u, d(t), d(k), d(p), d(m))
    want = nn.sample(x[:n], u, d(np.array([0, 0, 1, 1, 1, 1], np.float32)), 0, d(np.array([1, 1, 1, 1, 0, 1], np.float32)), d(np.array([0, 0, 0, 0, 0, 1], np.float32)))
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype,shift,stride", [("f32", 1, 4099), ("bf16", 1, 4099), ("bf16", 7, 4104), ("f32", 0, 0), ("bf16", 3, 0)])
def test_samples_of_strided_rows(gpu, dtype, shift, stride):
    torch = gpu
    rng = np.random.default_rng(7)
    flat = torch.from_numpy(logits(rng, 1, 12 * 4104)[0]).cuda().to(torch.float32 if dtype == "f32" else torch.bfloat16)
    x = flat.as_strided((11, 4090), (stride, 1), shift)
    for how in (dict(), dict(top_k=30, top_p=0.8), dict(top_p=0.99)):
        check_samples(torch, x, rng.random(11), **how)


def test_samples_of_the_largest_vocabulary_and_of_many_rows(gpu):
    torch = gpu
    from gomlx_amd import _lib, nn
    rng = np.random.default_rng(8)
    most = 2 ** 21 - 7
    x = torch.randn(1, most + 1, device="cuda")
    for how in (dict(), dict(top_k=40, top_p=0.9), dict(top_p=0.5)):
        check_samples(torch, x[:, :most], rng.random(1), **how)
        check_samples(torch, x[:, 1:], rng.random(1), **how)
    with pytest.raises(_lib.HipqError):
        nn.sample(x, torch.rand(1, device="cuda"))
    # more rows than the workspace holds at a time
    rows = 501000
    x, u = torch.randn(rows, 2, device="cuda"), torch.rand(rows, device="cuda")
    t = torch.rand(rows, device="cuda") + 0.5
    p = torch.exp((x.double() - x.double().amax(-1, keepdim=True)) / t.double()[:, None])
    share = p[:, 0] / p.sum(-1)
    fine = (share - u.double()).abs() > 1e-9
    assert torch.equal(nn.sample(x, u, t)[fine], (share <= u.double()).int()[fine])
    assert nn.sample(x[:0], u[:0]).shape == (0,)


def test_samples_replay_from_a_graph(gpu):
    torch = gpu
    from gomlx_amd import nn
    rng = np.random.default_rng(9)
    xs = [torch.from_numpy(logits(rng, 12, 20000, sure=i % 2 == 0)).cuda() for i in range(4)]
    us = [torch.rand(12, device="cuda") for _ in range(4)]
    x, u = xs[0].clone(), us[0].clone()
    call = lambda: nn.sample(x, u, 0.9, 0, 0.9, probabilities=True)  # noqa: E731
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        call()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = call()
    for i in (1, 2, 3, 0, 2):
        x.copy_(xs[i])
        u.copy_(us[i])
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graph.replay()
        eager = call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_sample_refuses(gpu):
    torch = gpu
    from gomlx_amd import _lib, nn
    x, u = torch.randn(3, 100, device="cuda"), torch.rand(3, device="cuda")
    nn.sample(x, u)
    for bad in (dict(logits=x[0]), dict(logits=x.cpu()), dict(logits=x[:, :0]), dict(logits=x.t()), dict(uniform=u[:2]), dict(uniform=u.double()), dict(uniform=u.cpu()), dict(temperature=-1.0),
                dict(top_k=-1), dict(top_p=1.5), dict(min_p=float("nan")), dict(top_k=u), dict(temperature=u[:2]), dict(top_p=u.cpu())):
        with pytest.raises(ValueError):
            nn.sample(**{**dict(logits=x, uniform=u), **bad})
    with pytest.raises(_lib.NotImplementedByBackend):
        nn.sample(x.half(), u)


@pytest.mark.parametrize("native", (True, False))
def test_sample_takes_whole_numbers_as_top_k(gpu, monkeypatch, native):
    torch = gpu
    from gomlx_amd import _lib, nn
    if not native:
        monkeypatch.setattr(_lib, "fast", None)
    x, u = torch.randn(40, 100, device="cuda"), torch.rand(40, device="cuda")
    for bad in (0.5, 2.9, 99.999, math.inf, math.nan, -0.5, np.float32(1.5)):
        with pytest.raises(ValueError, match="top_k"):
            nn.sample(x, u, top_k=bad)
    three, all_of_it = nn.sample(x, u, top_k=3), nn.sample(x, u)
    assert not torch.equal(three, all_of_it)
    for k in (3.0, np.int64(3), np.float32(3), torch.full((40,), 3, dtype=torch.int32, device="cuda")):
        assert torch.equal(nn.sample(x, u, top_k=k), three)
    for k in (0.0, 100, 2 ** 31 - 1, 2 ** 31, 2 ** 70):
        assert torch.equal(nn.sample(x, u, top_k=k), all_of_it)


# ---- the end of a step ----------------------------------------------------------------------------------------------------


def check_accept(c, news, parents, tokens, sampled, with_accounts=True, max_new=None, words=None):
    torch, nn = c.torch, c.nn
    max_new = max(news) if max_new is None else max_new
    accounts = torch.from_numpy(c.rng.random((c.pages, c.kv_heads, c.page)).astype(np.float32)).cuda() if with_accounts else None
    before, weights = c.host().copy(), None if accounts is None else accounts.cpu().numpy()
    single = max_new == 1
    flat = [ints(c.torch, sum((list(x) for x in v), [])) for v in (parents, tokens, sampled)]
    path, token, lengths = nn.kv_cache_accept(c.cache, c.d_table, c.ints(c.lengths), *flat, starts=None if single else c.ints(starts_of(news)), max_new=max_new, weights=accounts)
    after, at = c.host(), 0
    expect = None if weights is None else weights.copy()
    touched = np.zeros((c.pages, c.page // 32, 32), bool)
    for b, n in enumerate(news):
        want = ref.walk(parents[b], tokens[b], sampled[b])
        assert path[b].tolist() == want + [-1] * (max_new - len(want))
        assert token[b].item() == (sampled[b][want[-1]] if want else -1)
        first = c.lengths[b] - n
        new = first + len(want)
        assert lengths[b].item() == new
        places = np.concatenate([np.arange(first), first + np.array(want, int)]).astype(int)
        for h in range(c.kv_heads):
            for x, y in zip(kv_ref.decode(before, c.table[b], c.lengths[b], h), kv_ref.decode(after, c.table[b], new, h)):
                assert np.array_equal(x[places], y)
            if expect is not None:
                w = [weights[c.table[b, p // c.page], h, p % c.page] for p in places]
                for p in range(new):
                    expect[c.table[b, p // c.page], h, p % c.page] = w[p]
        for i, p in enumerate(range(first, new)):
            if want[i] != i:
                touched[c.table[b, p // c.page], p % c.page // 32, p % 32] = True
        at += n
    if expect is not None:
        assert np.array_equal(accounts.cpu().numpy(), expect)
    # nothing else has changed: tokens that are not the path's, other sequences' pages
    for p in range(c.pages):
        for t in range(c.page // 32):
            for h in range(c.kv_heads):
                for values in (False, True):
                    x, y = (kv_ref.decode_tile(z[p, h, t], values) for z in (before, after))
                    assert np.array_equal(x[~touched[p, t]], y[~touched[p, t]])


@pytest.mark.parametrize("dim", (64, 128, 256))
@pytest.mark.parametrize("news,lengths", [([1], [1]), ([1, 1], [33, 64]), ([16, 9, 30], [16, 100, 61]), ([70, 0, 33, 64], [200, 5, 33, 96])])
def test_accept_moves_the_path(gpu, dim, news, lengths):
    torch = gpu
    c = Case(torch, lengths, kv_heads=3, dim=dim, page=32, seed=dim + len(news)).fill()
    for bend in (0.3, 1.0, 3.0):  # chains, bushes
        parents = [random_parents(c.rng, n, bend) if n else [] for n in news]
        tokens = [c.rng.integers(0, 50, n).tolist() for n in news]
        sampled = []
        for p, t in zip(parents, tokens):
            children = [[j for j in range(len(p)) if p[j] == i] for i in range(len(p))]
            sampled.append([t[c.rng.choice(k)] if k and c.rng.random() < 0.9 else int(c.rng.integers(0, 50)) for k in children])
        check_accept(c, news, parents, tokens, sampled, with_accounts=bend != 1.0)


def test_accept_of_long_chains_and_late_children(gpu):
    """Paths of several tiles, whole and with every other node; children behind the first 64 rows."""
    torch = gpu
    for step, n in ((1, 150), (2, 150), (70, 211)):
        c = Case(torch, [n + 45, n], dim=64, page=32, seed=step).fill()
        parents = [[i - step if i >= step and i % step == 0 else -1 for i in range(n)] for _ in range(2)]
        tokens = [list(range(n)), list(range(n))]
        sampled = [[i + step for i in range(n)], [i + step if i < 100 else -1 for i in range(n)]]
        check_accept(c, [n, n], parents, tokens, sampled)


def test_accept_of_rows_that_are_not_there(gpu):
    """Rows in front of a sequence's first token, places behind the page table, pages that are none: their tokens are not moved, the answer is the walk's."""
    torch = gpu
    from gomlx_amd import nn
    c = Case(torch, [40, 64], kv_heads=1, dim=64, page=32, seed=1).fill()
    before = c.host().copy()
    up, word, drawn = [-1, 0, 0, 2, 3, 4], [0, 1, 2, 3, 4, 5], [2, 0, 3, 4, 5, 9]
    two = lambda v: ints(torch, v + v)  # noqa: E731
    starts = c.ints([0, 6, 12])
    # lengths that are shorter than the rows: row 0 at place -4
    path, token, lengths = nn.kv_cache_accept(c.cache, c.d_table, c.ints([2, 0]), two(up), two(word), two(drawn), starts=starts, max_new=6)
    assert path.tolist() == [[0, 2, 3, 4, 5, -1]] * 2 and token.tolist() == [9, 9] and lengths.tolist() == [1, 0]
    x, y = (kv_ref.decode(z, c.table[0], 40, 0) for z in (before, c.host()))
    for a, b in zip(x, y):
        assert np.array_equal(a[1], b[0]) and np.array_equal(a[1:], b[1:])
    # a table whose second page is none
    before = c.host().copy()
    table = c.table.copy()
    table[:, 1] = (-1, 10 ** 6)
    path, _, lengths = nn.kv_cache_accept(c.cache, torch.from_numpy(table).cuda(), c.ints([35, 35]), two(up), two(word), two(drawn), starts=starts, max_new=6)
    assert lengths.tolist() == [34, 34]
    x, y = (kv_ref.decode(z, c.table[0], 40, 0) for z in (before, c.host()))
    for a, b in zip(x, y):  # rows 0 to 5 at 29 to 34: of the path 31 has moved to 30; 32, 33 and 34 are not there
        assert np.array_equal(a[31], b[30]) and np.array_equal(np.delete(a, 30, 0), np.delete(b, 30, 0))


def test_accept_refuses(gpu):
    torch = gpu
    c = Case(torch, [40, 50]).fill()
    up, starts = ints(torch, [-1, 0, 0, -1, 0, 0, 1]), c.ints([0, 3, 7])
    good = dict(cache=c.cache, page_table=c.d_table, lengths=c.ints([40, 50]), parents=up, tokens=up, sampled=up, starts=starts, max_new=4)
    c.nn.kv_cache_accept(**good)
    for bad in (dict(parents=up.long()), dict(tokens=up[:6]), dict(sampled=up.cpu()), dict(parents=up.view(1, 7)), dict(max_new=0), dict(weights=torch.zeros(3, device="cuda")), dict(starts=None)):
        with pytest.raises(ValueError):
            c.nn.kv_cache_accept(**{**good, **bad})


# ---- together ---------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
def test_steps_with_drafts_leave_what_steps_without_leave(gpu, dtype):
    """Trees through two layers' caches, sampled and accepted, step after step, beside caches that get the accepted tokens one by one: the same keys and values, bit
    for bit, and at the accepted rows the same attention to the bound of both."""
    torch = gpu
    from gomlx_amd import nn
    rng = np.random.default_rng(11)
    seqs, layers, dim, kv_heads, heads, vocab = 3, 2, 64, 2, 8, 97
    t = torch.float32 if dtype == "f32" else torch.bfloat16
    table = torch.arange(seqs * 6, dtype=torch.int32, device="cuda").view(seqs, 6)
    drafted, plain = ([nn.kv_cache(seqs * 6, kv_heads, dim, 32) for _ in range(layers)] for _ in range(2))
    lengths, short = torch.zeros(seqs, dtype=torch.int32, device="cuda"), [0] * seqs
    head = torch.randn(heads * dim, vocab, device="cuda") * 0.3
    cos, sin = nn.rotary_table(300, dim)
    root = ints(torch, [1, 2, 3])
    for step in range(6):
        news = [int(n) for n in rng.integers(1, 14, seqs)]
        parents = [random_parents(rng, n, 1.5) for n in news]
        starts = ints(torch, starts_of(news))
        words = [rng.integers(0, vocab, n) for n in news]
        for b in range(seqs):
            words[b][0] = root[b].item()
        tokens = ints(torch, np.concatenate(words))
        rows = sum(news)
        kv = torch.randn(layers, 2, rows, kv_heads, dim, device="cuda").to(t)
        q = torch.randn(layers, rows, heads, dim, device="cuda").to(t)
        tree, positions = nn.draft_tree(ints(torch, sum(parents, [])), lengths, starts=starts, max_new=max(news))
        longer = lengths + ints(torch, news)
        outs, turned = [], []
        for n in range(layers):
            qr, kr = nn.qk_norm_rope(q[n], kv[n, 0], positions, cos, sin)
            turned.append((qr, kr))
            nn.kv_cache_append(drafted[n], kr, kv[n, 1], table, longer, starts=starts, max_new=max(news))
            outs.append(nn.tree_attention(qr, drafted[n], table, longer, tree, starts=starts, max_new=max(news)))
        drawn = nn.sample(outs[-1].float().view(rows, -1) @ head, torch.rand(rows, device="cuda"), temperature=0.5, top_k=3)
        # let the drafts be right more often than chance would have it: a child takes its parent's sample
        words, sampled = tokens.cpu().numpy(), drawn.cpu().numpy()
        for b, p in enumerate(parents):
            for i in range(1, news[b]):
                if rng.random() < 0.5:
                    words[starts[b] + i] = sampled[starts[b] + p[i]]
        answers = [nn.kv_cache_accept(drafted[n], table, longer, ints(torch, sum(parents, [])), ints(torch, words), drawn, starts=starts, max_new=max(news)) for n in range(layers)]
        assert all(torch.equal(x, y) for x, y in zip(*answers))
        path, root, lengths = answers[0]
        for b in range(seqs):
            want = ref.walk(parents[b], words[starts[b]:starts[b] + news[b]], sampled[starts[b]:starts[b] + news[b]])
            assert [p for p in path[b].tolist() if p >= 0] == want
            for i in want:
                short[b] += 1
                r = slice(int(starts[b]) + i, int(starts[b]) + i + 1)
                for n in range(layers):
                    one = ints(torch, [short[b]])
                    nn.kv_cache_append(plain[n], turned[n][1][r], kv[n, 1, r], table[b:b + 1], one)
                    single = nn.cached_attention(turned[n][0][r], plain[n], table[b:b + 1], one)
                    assert torch.allclose(single.float(), outs[n][r].float(), rtol=2 ** -7 if dtype == "bf16" else 0, atol=2e-3 if dtype == "bf16" else 1e-5)
        assert lengths.tolist() == short
        for n in range(layers):
            for b in range(seqs):
                how = dict(starts=ints(torch, [0, short[b]]), max_new=short[b], rows=short[b])
                for x, y in zip(*(nn.kv_cache_read(z[n], table[b:b + 1], lengths[b:b + 1].contiguous(), **how) for z in (drafted, plain))):
                    assert torch.equal(x, y)
    assert sum(short) > 6 * seqs  # (some drafts were accepted)


def _example():
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "drafted_decoding.py")
    spec = importlib.util.spec_from_file_location("drafted_decoding", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_example_takes_drafts_through_the_layer_as_single_tokens(gpu, monkeypatch):
    """A step's accepted rows against the same tokens one by one over the keys and values that the step has left in the cache (of its own a single token would write
    others: projections by other kernels differ enough to round some of their values to the next of 16).  Each way of the layer is within 1e-2 of its output's 2-norm by
    the projections' contract (four in a chain within 1e-3 of their rows' largest), two of them within 2e-2 of each other."""
    torch = gpu
    from gomlx_amd import nn
    ex = _example()
    model = ex.Model(200, 512, 8, 2, 768, seed=4, positions=200)
    drafts = ex.Drafts(3, (3, 2, 1))
    assert drafts.nodes == 16 and drafts.parents[:16].tolist() == [-1, 0, 0, 0, 1, 1, 2, 2, 3, 3, 4, 5, 6, 7, 8, 9]
    caches = ex.Caches(model.layer, 3, 150, 32)
    roots, seen = torch.tensor([5, 6, 7], dtype=torch.int32, device="cuda"), []
    forward = model.forward
    model.forward = lambda *a, **k: (seen.append((a[1], forward(*a, **k))), seen[-1][1])[1]
    for _ in range(8):
        before = caches.lengths.tolist()
        path, roots = ex.step(model, caches, drafts, roots, torch.rand(48, device="cuda"), temperature=0.0)
        tokens, h = seen.pop()
        assert path[:, 0].tolist() == [0, 0, 0]
        assert caches.lengths.tolist() == [n + int((p >= 0).sum()) for n, p in zip(before, path)]
        with monkeypatch.context() as m:
            m.setattr(nn, "kv_cache_append", lambda *a, **k: None)
            for b in range(3):
                one = ex.Caches.__new__(ex.Caches)
                one.data, one.table = caches.data, caches.table[b:b + 1]
                for i, node in enumerate(n for n in path[b].tolist() if n >= 0):
                    row, at = 16 * b + node, ints(torch, [before[b] + i])
                    single = forward(one, tokens[row:row + 1], at, at + 1, None, 1)
                    assert (single - h[row]).norm() <= 2e-2 * single.norm()


def test_example_runs(gpu, monkeypatch, capsys):
    ex = _example()
    monkeypatch.setattr("sys.argv", ["drafted_decoding.py", "--steps", "4", "--seqs", "3", "--prompt", "40", "--vocab", "300", "--shape", "512", "8", "2", "768"])
    ex.main()
    assert "tokens a sequence and step" in capsys.readouterr().out


def test_a_step_replays_from_a_graph(gpu):
    """Everything between the projections of a step, recorded once and replayed over other inputs with eager calls in between; some rows belong to no sequence."""
    torch = gpu
    from gomlx_amd import nn
    rng = np.random.default_rng(12)
    seqs, nodes, padding, heads, kv_heads, dim, vocab = 3, 9, 4, 8, 2, 64, 3000
    rows = seqs * nodes + padding
    table = torch.arange(seqs * 8, dtype=torch.int32, device="cuda").view(seqs, 8)
    starts = ints(torch, [0, 9, 18, 27])
    head = torch.randn(heads * dim, vocab, device="cuda")

    def inputs(seed):
        g = torch.Generator("cuda").manual_seed(seed)
        normal = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        parents = sum((random_parents(rng, nodes) for _ in range(seqs)), []) + [0] * padding
        return dict(lengths=ints(torch, [40 + seed, 9, 200 - seed]), parents=ints(torch, parents), tokens=ints(torch, rng.integers(0, 5, rows)), q=normal(rows, heads, dim), k=normal(rows, kv_heads, dim),
                    v=normal(rows, kv_heads, dim), u=torch.rand(rows, device="cuda", generator=g), cache=torch.randint(0, 100, (seqs * 8, kv_heads, 1, 36 * dim), dtype=torch.uint8, device="cuda", generator=g),
                    weights=normal(seqs * 8, kv_heads, 32).abs())

    def step(s):
        tree, positions = nn.draft_tree(s["parents"], s["lengths"], starts=starts, max_new=nodes)
        nn.kv_cache_append(s["cache"], s["k"], s["v"], table, s["lengths"], starts=starts, max_new=nodes, weights=s["weights"])
        a = nn.tree_attention(s["q"], s["cache"], table, s["lengths"], tree, starts=starts, max_new=nodes)
        drawn, shares = nn.sample(a.view(rows, -1) @ head, s["u"], 0.8, 0, 0.9, probabilities=True)
        path, token, lengths = nn.kv_cache_accept(s["cache"], table, s["lengths"], s["parents"], s["tokens"], drawn % 5, starts=starts, max_new=nodes, weights=s["weights"])
        real = slice(0, seqs * nodes)
        return [tree[real], positions[real], a[real], drawn[real], shares[real], path, token, lengths, s["cache"], s["weights"]]

    copy = lambda s: {k: t.clone() for k, t in s.items()}  # noqa: E731
    states = [inputs(i) for i in range(4)]
    held, stream = copy(states[0]), torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step(copy(states[0]))
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step(held)
    for i in (1, 2, 3, 0, 2):
        for k, t in states[i].items():
            held[k].copy_(t)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        eager = step(copy(states[i]))
        torch.cuda.synchronize()
        for n, (x, y) in enumerate(zip(out, eager)):
            assert torch.equal(x, y), f"state {i}, output {n}"


def test_attention_of_very_many_sequences(gpu):
    """Trees of a root alone are single new tokens."""
    torch = gpu
    from gomlx_amd import nn
    seqs = 9000
    cache = nn.kv_cache(seqs, 1, 64, 32)
    table = torch.randperm(seqs, device="cuda").int().view(seqs, 1)
    lengths = torch.randint(1, 33, (seqs,), dtype=torch.int32, device="cuda")
    starts = torch.cat([torch.zeros(1, device="cuda"), lengths.cumsum(0)]).int()
    rows = int(starts[-1])
    nn.kv_cache_append(cache, torch.randn(rows, 1, 64, device="cuda"), torch.randn(rows, 1, 64, device="cuda"), table, lengths, starts=starts, max_new=32)
    q = torch.randn(seqs, 4, 64, device="cuda")
    got = nn.tree_attention(q, cache, table, lengths, torch.ones(seqs, 1, dtype=torch.int32, device="cuda"))
    want = nn.cached_attention(q, cache, table, lengths)
    # (each within a few 2^-22 of 64 bits, times values of up to 5 that weights of 1 average)
    assert (got - want).abs().max() <= 1e-5


def test_calls_from_two_threads_on_streams_of_their_own(gpu):
    torch = gpu
    import threading
    from gomlx_amd import nn
    rng = np.random.default_rng(13)
    xs = [torch.from_numpy(logits(rng, 40, 30000, sure=i == 0)).cuda() for i in range(2)]
    us = [torch.rand(40, device="cuda") for _ in range(2)]
    cases = [Case(torch, [3000, 2000], seed=20 + i).fill() for i in range(2)]
    sets = [[ref.ancestors(random_parents(rng, 20)) for _ in range(2)] for _ in range(2)]
    trees = [torch.from_numpy(np.concatenate([ref.masks(s, 1) for s in ss])).cuda() for ss in sets]
    qs = [torch.randn(40, 8, 128, device="cuda") for _ in range(2)]

    def work(i):
        c = cases[i]
        return nn.sample(xs[i], us[i], 1.0, 0, 0.9), nn.tree_attention(qs[i], c.cache, c.d_table, c.ints([3000, 2000]), trees[i], starts=c.ints([0, 20, 40]), max_new=20)

    want = [work(i) for i in range(2)]
    torch.cuda.synchronize()
    bad = []

    def thread(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = work(i)
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(x, y) for x, y in zip(got, want[i])):
                    bad.append(i)

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_threads_finish_every_call(gpu):
    """Two threads at a time on streams of their own, and two on one stream: an error in a thread, or calls that it has not come to, fail the test as wrong results do."""
    torch = gpu
    import threading
    from gomlx_amd import nn
    rng = np.random.default_rng(19)
    calls, threads = 20, 4
    xs = [torch.from_numpy(logits(rng, 30, 30000, sure=i % 2 == 0)).cuda() for i in range(threads)]
    us = [torch.rand(30, device="cuda") for _ in range(threads)]
    cases = [Case(torch, [3000, 2000], seed=30 + i).fill() for i in range(threads)]
    caches = [c.cache.clone() for c in cases]
    parents = [[random_parents(rng, 20) for _ in range(2)] for _ in range(threads)]
    ups = [ints(torch, sum(p, [])) for p in parents]
    words = [ints(torch, rng.integers(0, 4, 40)) for _ in range(threads)]
    qs = [torch.randn(40, 8, 128, device="cuda") for _ in range(threads)]
    lengths, starts = ints(torch, [3000, 2000]), ints(torch, [0, 20, 40])

    def work(i):
        caches[i].copy_(cases[i].cache)
        tree, positions = nn.draft_tree(ups[i], lengths, starts=starts, max_new=20)
        out = nn.tree_attention(qs[i], caches[i], cases[i].d_table, lengths, tree, starts=starts, max_new=20)
        drawn, shares = nn.sample(xs[i], us[i], 1.0, 0, 0.9, probabilities=True)
        path, token, left = nn.kv_cache_accept(caches[i], cases[i].d_table, lengths, ups[i], words[i], words[i], starts=starts, max_new=20)
        return tree, positions, out, drawn, shares, path, token, left, caches[i].clone()

    want = [work(i) for i in range(threads)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    streams.append(streams[1])
    streams.append(torch.cuda.Stream())
    done, errors = [0] * threads, []

    def thread(i):
        try:
            with torch.cuda.stream(streams[i]):
                for _ in range(calls):
                    got = work(i)
                    streams[i].synchronize()
                    assert all(torch.equal(x, y) for x, y in zip(got, want[i])), f"thread {i}, call {done[i]}"
                    done[i] += 1
        except BaseException as e:  # noqa: BLE001 (a thread's own traceback is only printed)
            errors.append(e)

    running = [threading.Thread(target=thread, args=(i,)) for i in range(threads)]
    for t in running:
        t.start()
    for t in running:
        t.join()
    assert not errors, errors
    assert done == [calls] * threads


def test_native_host_path(gpu, monkeypatch):
    """The native steps serve the calls of a step with drafts, with the Python steps' results; what they do not know they leave alone."""
    torch = gpu
    from gomlx_amd import _lib, nn
    rng = np.random.default_rng(20)
    c = Case(torch, [90, 33], 2, 64, 32, seed=21, wide_table=1).fill()
    n, starts = c.ints([90, 33]), c.ints([0, 6, 11])
    up = ints(torch, random_parents(rng, 6) + random_parents(rng, 5))
    words, drawn = ints(torch, rng.integers(0, 3, 11)), ints(torch, rng.integers(0, 3, 11))
    q = torch.randn(11, 4, 64, device="cuda")
    x, u = torch.randn(11, 3000, device="cuda"), torch.rand(11, device="cuda")
    t, k = torch.rand(11, device="cuda"), ints(torch, rng.integers(0, 60, 11))
    p, m = torch.rand(11, device="cuda"), 0.1 * torch.rand(11, device="cuda")
    fast = _lib.fast
    assert fast is not None

    def calls():
        cache, w = c.cache.clone(), torch.arange(c.pages * 2 * 32, device="cuda").float().view(c.pages, 2, 32)
        tree, positions = nn.draft_tree(up, n, starts=starts, max_new=6)
        out = [tree, positions, *nn.draft_tree(up[:2].contiguous(), n)]
        out.append(nn.tree_attention(q, cache, c.d_table, n, tree, starts=starts, max_new=6))
        out.append(nn.tree_attention(q.bfloat16(), cache, c.d_table, n, tree, starts, 6, 0.3, 9))
        out.append(nn.tree_attention(q[:2], cache, c.d_table, n, tree[:2]))
        for y in (x, x.bfloat16(), x[:, 1:2990]):
            out += [nn.sample(y, u), nn.sample(y, u, 0), *nn.sample(y, u, 0.7, 40, 0.9, 0.01, True), *nn.sample(y, u, t, k, p, m, probabilities=True), nn.sample(y, u, t, 5, p)]
        out += [*nn.kv_cache_accept(cache, c.d_table, n, up, words, drawn, starts=starts, max_new=6, weights=w), cache.clone(), w]
        out += [*nn.kv_cache_accept(cache, c.d_table, n, up[:2].contiguous(), words[:2].contiguous(), drawn[:2].contiguous()), cache]
        return out

    native = calls()
    served = []

    class Spy:
        def __getattr__(self, name):
            def call(*args):
                result = getattr(fast, name)(*args)
                served.append((name, result is not None))
                return result
            return call

    monkeypatch.setattr(_lib, "fast", Spy())
    spied = calls()
    assert all(ok for _, ok in served) and {name for name, _ in served} == {"draft_tree", "tree_attention", "sample", "kv_accept"}
    monkeypatch.setattr(_lib, "fast", None)
    plain = calls()
    assert len(native) == len(plain) == len(spied)
    for a, b, d in zip(native, plain, spied):
        assert torch.equal(a, b) and torch.equal(a, d) and a.dtype == b.dtype and a.stride() == b.stride() and a.device == b.device
    tree = native[0]
    attend, accept = (q, c.cache, c.d_table, n, tree, starts, 6, None, 0), (c.cache, c.d_table, n, up, words, drawn, starts, 6, None)
    change = lambda args, i, v: args[:i] + (v,) + args[i + 1:]  # noqa: E731
    for f, args in ((fast.draft_tree, (up.long(), n, starts, 6)), (fast.draft_tree, (up, n[:1], starts, 6)), (fast.draft_tree, (up, n, None, 6)), (fast.draft_tree, (up, n, starts, 0)), (fast.draft_tree, (up.cpu(), n, starts, 6)),
                    (fast.tree_attention, change(attend, 0, q.half())), (fast.tree_attention, change(attend, 0, q[:, :3])), (fast.tree_attention, change(attend, 4, tree.long())),
                    (fast.tree_attention, change(attend, 4, tree[:10])), (fast.tree_attention, change(attend, 4, tree[:, :0])), (fast.tree_attention, change(attend, 8, -1)),
                    (fast.tree_attention, change(attend, 0, q.cpu())), (fast.sample, (x, u, 1.0, 0.5, 1.0, 0.0, False)), (fast.sample, (x, u, -1.0, 0, 1.0, 0.0, False)), (fast.sample, (x, u, 1.0, 0, 1.5, 0.0, False)),
                    (fast.sample, (x, u[:3], 1.0, 0, 1.0, 0.0, False)), (fast.sample, (x.half(), u, 1.0, 0, 1.0, 0.0, False)), (fast.sample, (x, u, 1.0, t, 1.0, 0.0, False)), (fast.sample, (x, u, t[:4], 0, 1.0, 0.0, False)),
                    (fast.sample, (x.t(), u, 1.0, 0, 1.0, 0.0, False)), (fast.kv_accept, change(accept, 4, words.long())), (fast.kv_accept, change(accept, 5, drawn[:10])), (fast.kv_accept, change(accept, 3, up.view(1, 11))),
                    (fast.kv_accept, change(accept, 7, 0)), (fast.kv_accept, change(accept, 6, None))):
        assert f(*args) is None


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("window", (0, 6))
@pytest.mark.parametrize("more", (1, 2, 9))
def test_attention_with_masks_wider_than_needed(gpu, dtype, window, more):
    """Words behind those that the largest tree needs, some with bits set: they count for nothing."""
    torch = gpu
    c = Case(torch, [130, 40, 31], dim=64, page=32, seed=22).fill()
    news = [33, 9, 31]
    words = 2 + more
    sets = [ref.ancestors(random_parents(c.rng, n)) for n in news]
    for s in sets:
        for row in s:
            row.update(int(j) for j in c.rng.choice(np.arange(66, 32 * words), 5, replace=False))
    check_attention(c, news, 8, sets, dtype, window=window, words=words)
