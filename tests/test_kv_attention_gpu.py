"""The operators between a layer's q / k / v projections and its output projection on the GPU, against their definition in 64 bits
(oracle/kv_oracle.py).  Tolerances are bounds that follow from the formats: see attention_bound() and rope_bound()."""
import numpy as np
import pytest

from oracle import kv_oracle as ref

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24  # half a unit of float32


class Case:
    """Sequences over a cache with scattered pages, filled by kv_cache_append in pieces."""

    def __init__(self, torch, lengths, kv_heads=2, dim=128, page=64, seed=0, wide_table=0, scale=1.0):
        from gomlx_amd import nn
        self.torch, self.nn, self.lengths, self.page, self.kv_heads, self.dim = torch, nn, lengths, page, kv_heads, dim
        self.rng = np.random.default_rng(seed)
        counts = [-(-n // page) for n in lengths]
        self.pages = sum(counts) + 2
        order = list(self.rng.permutation(self.pages))
        self.table = np.full((len(lengths), max(counts + [1]) + wide_table), -1, np.int32)
        for b, n in enumerate(counts):
            self.table[b, :n] = [order.pop() for _ in range(n)]
        self.cache = nn.kv_cache(self.pages, kv_heads, dim, page)
        self.d_table = torch.from_numpy(self.table).cuda()
        self.k = [(scale * self.rng.standard_normal((n, kv_heads, dim))).astype(np.float32) for n in lengths]
        self.v = [self.rng.standard_normal((n, kv_heads, dim)).astype(np.float32) for n in lengths]

    def ints(self, v):
        return self.torch.tensor(v, dtype=self.torch.int32, device="cuda")

    def fill(self, accounts=None):
        """Everything in one ragged call."""
        starts = np.concatenate([[0], np.cumsum(self.lengths)])
        if starts[-1]:
            k, v = (self.torch.from_numpy(np.concatenate(x)).cuda() for x in (self.k, self.v))
            self.nn.kv_cache_append(self.cache, k, v, self.d_table, self.ints(self.lengths), starts=self.ints(starts), max_new=max(self.lengths), weights=accounts)
        return self

    def host(self):
        return self.cache.cpu().numpy()

    def attend(self, news, heads, dtype="f32", window=0, accounts=None, q=None, scale=None, table=None):
        """(q rows float64, output) of a call with `news` new tokens of each sequence."""
        torch = self.torch
        rows = sum(news)
        if q is None:
            q = torch.from_numpy(self.rng.standard_normal((rows, heads, self.dim)).astype(np.float32)).cuda()
        q = q.to({"f32": torch.float32, "bf16": torch.bfloat16}[dtype])
        single = all(n == 1 for n in news)
        starts = None if single else self.ints(np.concatenate([[0], np.cumsum(news)]))
        out = self.nn.cached_attention(q, self.cache, self.d_table if table is None else table, self.ints(self.lengths), starts=starts,
                                       max_new=1 if single else max(news), window=window, weights=accounts, scale=scale)
        assert out.dtype == q.dtype and out.shape == q.shape and out.is_contiguous()
        return q.double().cpu().numpy(), out.double().cpu().numpy()

    def check(self, news, heads, dtype="f32", window=0, with_accounts=False, q=None, scale=None):
        torch, group = self.torch, heads // self.kv_heads
        accounts = before = None
        if with_accounts:
            before = self.rng.random((self.pages, self.kv_heads, self.page)).astype(np.float32)
            accounts = torch.from_numpy(before.copy()).cuda()
        q, out = self.attend(news, heads, dtype, window, accounts, q, scale)
        host, at = self.host(), 0
        scale = self.dim ** -0.5 if scale is None else scale
        expect = None if before is None else before.astype(np.float64)
        slack = None if before is None else np.abs(expect) * 2 * EPS
        for b, n in enumerate(news):
            for h in range(self.kv_heads):
                keys, values = ref.decode(host, self.table[b], self.lengths[b], h)
                qb = q[at:at + n, h * group:(h + 1) * group]
                want, p, s, seen = ref.attention(qb, keys, values, scale, window)
                got = out[at:at + n, h * group:(h + 1) * group]
                if n and not seen.any(-1).all():
                    assert np.all(got[~seen.any(-1)] == 0)
                bound, eps_p = attention_bound(qb, keys, values, scale, p, s, seen, dtype)
                bad = np.isnan(want).any(-1)
                assert np.isnan(got[bad]).all()
                assert np.all(np.abs(got - want)[~bad] <= (bound + np.abs(want) * (2.0 ** -8 if dtype == "bf16" else 2 * EPS))[~bad]), \
                    f"sequence {b}, head {h}: {np.max((np.abs(got - want) - bound)[~bad])}"
                if expect is not None:
                    for t in range(self.lengths[b]):
                        add = p[:, :, t][np.broadcast_to(seen[:, None, t], p.shape[:2])]
                        w = (self.table[b, t // self.page], h, t % self.page)
                        expect[w] += add.sum()
                        slack[w] += (np.abs(add) * (np.broadcast_to(eps_p, p.shape[:2])[np.broadcast_to(seen[:, None, t], p.shape[:2])] + (add.size + 4) * EPS)).sum() + expect[w] * EPS
            at += n
        if expect is not None:
            got = accounts.cpu().numpy().astype(np.float64)
            assert np.all(np.isnan(got) == np.isnan(expect))
            fine = ~np.isnan(expect)
            assert np.all(np.abs(got - expect)[fine] <= slack[fine]), np.max((np.abs(got - expect) - slack)[fine])
        return out


def attention_bound(q, keys, values, scale, p, s, seen, dtype):
    """Largest error of a row's results before the rounding of the output, and relative error of its weights.

    q is used to 2^-22 of its row's largest value (float32; bfloat16 exactly), products are exact, a score is a sum of D of them in
    float32 and scaled: |ds| <= scale (2^-22 + D 2^-24) max_j sum_d max|q| |k_jd| + 2^-22 max|s|.  exp2 adds 2^-22.  A softmax weight is
    then off by a factor of at most 1 + 2 (|ds| + 2^-22) (the sum's error included), plus n 2^-24 of the sum's additions.  As operands weights are rounded to 2^-22 (float32) or 2^-12
    (bfloat16) of themselves or, where tiny, 2^-30 of the largest.  n additions in float32 in the second product."""
    n = keys.shape[0]
    if n == 0 or q.size == 0:
        return np.zeros(q.shape), np.zeros(q.shape[:2])
    with np.errstate(all="ignore"):
        k = np.nan_to_num(np.abs(keys))
        qk = np.abs(q).max(-1) * max(k.sum(-1).max(), 0)
        top = np.max(np.where(np.isfinite(s), np.abs(s), 0), -1)
        ds = scale * (2.0 ** -22 + q.shape[-1] * EPS) * qk + 2.0 ** -22 * top
        eps_p = 2 * (ds + 2.0 ** -22) + n * EPS
        operand = 2.0 ** -12 if dtype == "bf16" else 2.0 ** -22
        size = np.einsum("ngt,td->ngd", np.nan_to_num(p), np.abs(values))
        bound = (eps_p + operand + (n + 8) * EPS)[..., None] * size + n * 2.0 ** -30 * np.abs(values).max(initial=0)
    return bound, eps_p


# ---- the cache --------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dim", (64, 128, 256))
@pytest.mark.parametrize("dtype", ("f32", "bf16"))
def test_append_holds_what_the_definition_says(gpu, dim, dtype):
    """Bit for bit, in one ragged call, token by token, and from strided rows that no vector load fits."""
    torch = gpu
    lengths = [1, 7, 33, 100, 65]
    c = Case(torch, lengths, kv_heads=3, dim=dim, page=32)
    c.k[3][5, 1] = 0.0                                        # a head of zeros
    c.k[3][6, 0, :32] = 1e-7                                  # a scale below fp16's smallest
    c.v[3][7, 2, 3], c.v[3][7, 2, 9] = 4.0, -4.0              # a tie: the first one's sign
    c.k[4][0] = 60000.0 * np.sign(c.k[4][0])                  # near the largest scale
    if dtype == "bf16":
        c.k, c.v = ([torch.from_numpy(x).bfloat16().float().numpy() for x in y] for y in (c.k, c.v))
    c.fill()
    want = [ref.quantise(k, v) for k, v in zip(c.k, c.v)]
    starts = np.concatenate([[0], np.cumsum(lengths)])

    def same(cache):
        k, v = c.nn.kv_cache_read(cache, c.d_table, c.ints(lengths), starts=c.ints(starts), max_new=100, rows=int(starts[-1]))
        for got, which in ((k, 0), (v, 1)):
            got = got.double().cpu().numpy()
            for b in range(len(lengths)):
                assert np.array_equal(got[starts[b]:starts[b + 1]], want[b][which])

    same(c.cache)
    host = c.host()
    for b, n in enumerate(lengths):  # the bytes themselves
        for h in range(3):
            k, v = ref.decode(host, c.table[b], n, h)
            assert np.array_equal(k, want[b][0][:, h]) and np.array_equal(v, want[b][1][:, h])
    kind = {"f32": torch.float32, "bf16": torch.bfloat16}[dtype]
    # token by token: sequences that still grow get one row each
    again = c.nn.kv_cache(c.pages, 3, dim, 32)
    wide = torch.zeros(len(lengths), 3 * (2 * dim + 3) + 1, dtype=kind, device="cuda")[:, 1:]  # rows and heads off every vector
    k, v = (wide.as_strided((len(lengths), 3, dim), (wide.stride(0), 2 * dim + 3, 1), wide.storage_offset() + o) for o in (0, dim + 1))
    for step in range(max(lengths)):
        now = [min(step + 1, n) for n in lengths]
        for b, n in enumerate(now):
            k[b], v[b] = torch.from_numpy(c.k[b][n - 1]).cuda().to(kind), torch.from_numpy(c.v[b][n - 1]).cuda().to(kind)
        c.nn.kv_cache_append(again, k, v, c.d_table, c.ints(now))
    same(again)


def test_append_in_pieces_keeps_the_neighbours(gpu):
    """Pieces that begin and end inside a block of eight tokens, a tile and a page leave every other token as it was, and stay inside
    the pages of their sequence."""
    c = Case(gpu, [200, 90], kv_heads=2, dim=64, page=64, seed=3)
    c.cache.random_(0, 256)
    before = c.host().copy()
    done = [0, 0]
    for pieces in ([5, 3], [1, 1], [60, 29], [64, 0], [70, 57]):
        done = [a + n for a, n in zip(done, pieces)]
        starts = np.concatenate([[0], np.cumsum(pieces)])
        k, v = (gpu.from_numpy(np.concatenate([x[b][done[b] - n:done[b]] for b, n in enumerate(pieces)])).cuda() for x in (c.k, c.v))
        c.nn.kv_cache_append(c.cache, k, v, c.d_table, c.ints(done), starts=c.ints(starts), max_new=max(pieces))
    host = c.host()
    for b, n in enumerate(c.lengths):
        want = ref.quantise(c.k[b], c.v[b])
        for h in range(2):
            k, v = ref.decode(host, c.table[b], n, h)
            assert np.array_equal(k, want[0][:, h]) and np.array_equal(v, want[1][:, h])
            # behind the last token: as before
            whole = -(-n // 64) * 64
            old, new = (ref.decode(x, c.table[b], whole, h) for x in (before, host))
            for i in (0, 1):
                assert np.array_equal(old[i][n:], new[i][n:], equal_nan=True)
    free = sorted(set(range(c.pages)) - set(c.table[c.table >= 0].tolist()))
    assert free and np.array_equal(before[free], host[free])


def test_append_bad_tokens_and_accounts(gpu):
    c = Case(gpu, [40], kv_heads=2, dim=128, page=64)
    c.k[0][3, 0, 5] = np.nan
    c.v[0][9, 1, 127] = np.inf
    c.k[0][11, 1, 64] = 65408.0
    c.v[0][12, 0, 0] = -65407.0
    accounts = gpu.ones(c.pages, 2, 64, device="cuda")
    c.fill(accounts)
    host = c.host()
    want = ref.quantise(c.k[0], c.v[0])
    for h in range(2):
        k, v = ref.decode(host, c.table[0], 40, h)
        assert np.array_equal(k, want[0][:, h], equal_nan=True) and np.array_equal(v, want[1][:, h])
    assert np.isnan(want[0]).all(-1).sum() == 3
    got = accounts.cpu().numpy()
    assert np.all(got[c.table[0, 0], :, :40] == 0) and got.sum() == got.size - 80


def test_read_in_front_of_the_first_token_and_absent_pages(gpu):
    c = Case(gpu, [5, 70], kv_heads=1, dim=64, page=32).fill()
    c.d_table[1, 1] = c.pages  # tokens 32 to 63 of the second sequence have no page
    k, v = c.nn.kv_cache_read(c.cache, c.d_table, c.ints([5, 70]), starts=c.ints([0, 12, 90]), max_new=78, rows=90)
    k, v = k.double().cpu().numpy(), v.double().cpu().numpy()
    w0, w1 = ref.quantise(c.k[0], c.v[0]), ref.quantise(c.k[1], c.v[1])
    for got, i in ((k, 0), (v, 1)):
        assert np.all(got[:7] == 0) and np.array_equal(got[7:12], w0[i])
        assert np.all(got[12:20] == 0) and np.array_equal(got[20:52], w1[i][:32]) and np.all(got[52:84] == 0) and np.array_equal(got[84:], w1[i][64:])


@pytest.mark.parametrize("dim", (64, 128, 256))
@pytest.mark.parametrize("dtype", ("f32", "bf16"))
def test_one_prompt_beside_many_sequences(gpu, dim, dtype):
    """A call whose sequences differ widely in new tokens, none among them, some of more rows than tokens and some past their page table: every token lies where it belongs,
    and is read back."""
    torch = gpu
    rng = np.random.default_rng(dim)
    news = [int(n) for n in rng.integers(0, 3, 200)]
    news[70], news[131], news[199] = 700, 33, 5
    room = 768
    lengths = [n + int(x) for n, x in zip(news, rng.integers(0, 60, 200))]
    lengths[131], lengths[199], lengths[3] = 20, room + 2, 0
    news[3] = 2
    c = Case(torch, [min(n, room) for n in lengths], 2, dim, 96, seed=dim)
    assert c.table.shape[1] * 96 == room
    rows, starts = sum(news), np.concatenate([[0], np.cumsum(news)])
    k, v = (torch.from_numpy(rng.standard_normal((rows, 2, dim)).astype(np.float32)).cuda().to({"f32": torch.float32, "bf16": torch.bfloat16}[dtype]) for _ in range(2))
    accounts = torch.ones(c.pages, 2, 96, device="cuda")
    how = dict(starts=c.ints(starts), max_new=700)
    c.nn.kv_cache_append(c.cache, k, v, c.d_table, c.ints(lengths), weights=accounts, **how)
    want = ref.quantise(k.float().cpu().numpy(), v.float().cpu().numpy())
    got = [x.double().cpu().numpy() for x in c.nn.kv_cache_read(c.cache, c.d_table, c.ints(lengths), rows=rows, **how)]
    host, left = c.host(), np.ones((c.pages, 2, 96), np.float32)
    for b, n in enumerate(news):
        place = np.arange(lengths[b] - n, lengths[b])
        there = (place >= 0) & (place < room)
        for h in range(2):
            for i, x in enumerate(ref.decode(host, c.table[b], min(lengths[b], room), h)):
                new = want[i][starts[b]:starts[b + 1], h]
                assert np.array_equal(x[place[there]], new[there])
                assert np.array_equal(got[i][starts[b]:starts[b + 1], h], np.where(there[:, None], new, 0))
        left[c.table[b, place[there] // 96], :, place[there] % 96] = 0
    assert np.array_equal(accounts.cpu().numpy(), left)


def test_a_very_long_prompt_beside_many_single_tokens(gpu):
    """131072 new tokens of one sequence and one of each of 511: more blocks of eight tokens a sequence, key head and sequences than a launch has threads for."""
    torch = gpu
    from gomlx_amd import nn
    n, others, heads, dim, page = 131072, 511, 8, 64, 256
    k, v = (torch.randn(n + others, heads, dim, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    table = torch.full((others + 1, n // page), -1, dtype=torch.int32, device="cuda")
    table[200] = torch.arange(n // page, dtype=torch.int32, device="cuda")
    rest = [b for b in range(others + 1) if b != 200]
    table[rest, 0] = torch.arange(n // page, n // page + others, dtype=torch.int32, device="cuda")
    lengths = torch.full((others + 1,), 9, dtype=torch.int32, device="cuda")
    lengths[200] = n
    starts = torch.tensor([b if b <= 200 else b + n - 1 for b in range(others + 2)], dtype=torch.int32, device="cuda")
    caches = [nn.kv_cache(n // page + others, heads, dim, page) for _ in range(2)]
    nn.kv_cache_append(caches[0], k, v, table, lengths, starts=starts, max_new=n)
    nn.kv_cache_append(caches[1], k[200:200 + n], v[200:200 + n], table[200:201], lengths[200:201], starts=torch.tensor([0, n], dtype=torch.int32, device="cuda"), max_new=n)
    single = [torch.cat([x[:200], x[200 + n:]]) for x in (k, v)]
    nn.kv_cache_append(caches[1], *single, table[rest].contiguous(), lengths[rest].contiguous())
    assert torch.equal(*caches)
    got = nn.kv_cache_read(caches[0], table, lengths, starts=starts, max_new=n, rows=n + others)
    want = nn.kv_cache_read(caches[0], table[200:201], lengths[200:201], starts=torch.tensor([0, n], dtype=torch.int32, device="cuda"), max_new=n, rows=n)
    alone = nn.kv_cache_read(caches[0], table[rest].contiguous(), lengths[rest].contiguous())
    for x, y, z in zip(got, want, alone):
        assert torch.equal(x[200:200 + n], y) and torch.equal(torch.cat([x[:200], x[200 + n:]]), z)


# ---- attention --------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("dim,kv_heads,heads,page", ((64, 3, 3, 32), (128, 2, 8, 64), (128, 1, 7, 96), (256, 2, 4, 32), (64, 1, 40, 64)))
def test_single_tokens(gpu, dtype, dim, kv_heads, heads, page):
    """Lengths around tiles and pages, from nothing to several workgroups' worth."""
    c = Case(gpu, [1, 0, 31, 32, 33, 64, 65, 500, 1285], kv_heads, dim, page, seed=dim + heads).fill()
    c.check([1] * 9, heads, dtype, with_accounts=True)
    c.check([1] * 9, heads, dtype, window=40, with_accounts=True)


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("dim,kv_heads,heads,window", ((128, 2, 8, 0), (64, 2, 2, 0), (256, 1, 3, 0), (128, 1, 4, 33), (64, 1, 5, 1), (256, 2, 4, 100)))
def test_several_tokens(gpu, dtype, dim, kv_heads, heads, window):
    """Ragged prompts on top of caches, sequences without a new token, prompts that are the whole cache."""
    c = Case(gpu, [300, 70, 129, 1, 64], kv_heads, dim, 64, seed=window + heads).fill()
    c.check([3, 70, 0, 1, 40], heads, dtype, window, with_accounts=True)
    c.check([131, 17, 129, 1, 5], heads, dtype, window, with_accounts=True)


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("dim,heads,window", ((64, 8, 0), (128, 8, 0), (256, 8, 0), (128, 2, 700), (64, 32, 50)))
def test_prompts_beside_single_tokens(gpu, dtype, dim, heads, window):
    """One call whose sequences differ in new tokens, so that some have few rows over many tokens and some many: at two key heads of `heads` queries,
    5 and 4 new tokens lie on either side of sixteen rows."""
    c = Case(gpu, [2100, 300, 40, 1000, 33, 1, 900] + [5] * 40, dim=dim, page=96, seed=dim + heads, wide_table=30).fill()
    c.check([1, 70, 0, 4, 5, 1, 3] + [1] * 40, heads, dtype, window, with_accounts=True)
    c.check([2, 0, 1, 1, 1, 0, 45] + [0, 1] * 20, heads, dtype, window)


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("heads", (17, 40))
def test_prompts_beside_single_tokens_at_many_heads_a_key_head(gpu, dtype, heads):
    """More than sixteen query heads a key head: single tokens are many rows as well, and no launch goes out for sequences of few."""
    torch = gpu
    import ctypes
    from gomlx_amd import _lib
    c = Case(torch, [900, 300, 40, 700] + [9] * 30, kv_heads=1, dim=64, page=64, seed=heads, wide_table=30).fill()
    news = [1, 70, 0, 2] + [1] * 30
    c.check(news, heads, dtype, with_accounts=True)
    c.check(news, heads, dtype, window=33)
    for accounts in (None, torch.zeros(c.pages, 1, 64, device="cuda")):
        launches = ctypes.c_int()
        _lib.check(_lib.lib().gq_profile_begin())
        c.attend(news, heads, dtype, accounts=accounts)
        _lib.check(_lib.lib().gq_profile_end(ctypes.byref(launches), None))
        assert launches.value <= (2 if accounts is None else 3)


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("dim", (64, 128, 256))
def test_accounts_where_scores_have_no_room(gpu, dtype, dim):
    """A page table of 15000 columns: the scores of the rows that it has room for would be more than 256 MB, so the accounts are made from the keys."""
    c = Case(gpu, [1, 0, 33, 500, 64, 130, 31, 90, 700], 2, dim, 64, seed=dim, wide_table=15000).fill()
    c.check([1] * 9, 8, dtype, with_accounts=True)
    c.check([1, 0, 2, 4, 3, 1, 1, 4, 2], 6, dtype, with_accounts=True)


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
def test_prompt_of_a_thousand_tokens(gpu, dtype):
    c = Case(gpu, [1217], 1, 128, 128, seed=9).fill()
    c.check([1001], 4, dtype, with_accounts=True)
    c.check([1001], 4, dtype, window=300)


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("news", (1, 40))
def test_large_and_small_scores(gpu, dtype, news):
    """Softmax from nearly one token to nearly flat, large queries and tiny ones, and a scale of the caller's."""
    c = Case(gpu, [400], 2, 128, 64, seed=4, scale=3.0).fill()
    q = gpu.randn(news, 4, 128, device="cuda", generator=gpu.Generator("cuda").manual_seed(1))
    for factor in (1e-30, 1e-4, 1.0, 30.0):
        c.check([news], 4, dtype, q=q * factor)
    c.check([news], 4, dtype, q=q, scale=0.7)
    c.check([news], 4, dtype, q=q * 1e30, scale=1e-31)
    c.check([news], 4, dtype, q=q, scale=0.0, with_accounts=True)


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("dim,news", ((64, 1), (64, 40), (256, 1), (256, 40), (256, 130)))
def test_scores_that_grow_along_the_sequence(gpu, dtype, dim, news):
    """What a row has summed is scaled down again and again: later keys are larger, and queries so large that every tile has a new largest score."""
    c = Case(gpu, [420], 2, dim, 64, seed=dim + news, scale=2.0)
    c.k[0] *= np.linspace(0.1, 1.5, 420, dtype=np.float32)[:, None, None]
    c.fill()
    q = gpu.randn(news, 4, dim, device="cuda", generator=gpu.Generator("cuda").manual_seed(news))
    for factor in (2.0, 25.0):
        c.check([news], 4, dtype, q=q * factor, with_accounts=True)


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("dim", (64, 128, 256))
@pytest.mark.parametrize("news", (1, 40))
def test_scores_past_the_whole_numbers_of_float32(gpu, dtype, dim, news):
    """Scores of 10^4 to 10^23, whose rounding in float32 is far more than the room of an exponent: the largest takes all the weight.  (Keys are
    multiples of a vector of ones, so that scores are the exact products of few bits, rounded with the scale alone.)"""
    torch = gpu
    c = Case(torch, [300], 2, dim, 64, seed=dim)
    c.k[0][:] = (1 + np.arange(300) % 7 / 8).astype(np.float32)[:, None, None]
    c.k[0][33] = 2.0
    c.fill()
    q = torch.ones(news, 4, dim, device="cuda")
    value = np.stack([ref.decode(c.host(), c.table[0], 300, h)[1][33] for h in (0, 0, 1, 1)])
    weights = np.zeros((c.pages, 2, 64))
    weights[c.table[0, 0], :, 33] = 2 * news
    for scale in (100.0, 3e3, 1e5, 7.7e5, 3e6, 1.23e7, 1e8, 3.3e9, 1e12, 1.7e20, -1e8):
        got = torch.zeros(c.pages, 2, 64, device="cuda")
        sign = -1 if scale < 0 else 1
        _, out = c.attend([news], 4, dtype, q=sign * q, scale=scale, accounts=got)
        _, again = c.attend([news], 4, dtype, q=sign * q, scale=scale)
        for y in (out, again):  # the weight's rounding as an operand (its sum may be of unrounded ones) and the output's
            assert np.all(np.abs(y - value) <= np.abs(value) * (2.0 ** -8 + 2.0 ** -10 if dtype == "bf16" else 2.0 ** -20)), scale
        # a weight of one: the sum's logarithm is rounded as the score is, and both are equal but for that
        assert np.all(np.abs(got.cpu().numpy() - weights) <= weights * 2.0 ** -6), scale


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("dim", (64, 128, 256))
@pytest.mark.parametrize("news", (1, 9, 70, 4200))
@pytest.mark.parametrize("accounts", (False, True))
def test_one_large_weight_beside_many_small_ones(gpu, dtype, dim, news, accounts):
    """60000 tokens, of which the first has 2^18 to 2^36 times the weight of every other: what these add up to is not lost.  The first one's value is 0 and
    the others' 1, so that a result is the others' share.  A weight is off by 2^-31 (bfloat16) or 2^-37 (float32; 2^-34 at head_dim 256) of the row's largest at most, half
    the spacing of the smallest operands, beside the relative errors: of sixty thousand additions in float32, of the exponent, of the output."""
    torch = gpu
    n = 60000
    c = Case(torch, [n], 1, dim, 256, seed=news)
    c.k[0][:], c.v[0][:] = 0.0, 1.0
    c.k[0][0], c.v[0][0] = 1.0, 0.0
    c.fill()
    heads = 8 if news == 4200 else 2  # (4200 rows of 8 heads: every row goes over all the tokens in one piece)
    q = torch.ones(news, heads, dim, device="cuda")
    others = np.arange(n - news, n, dtype=np.float64)  # in front of a row's own token, and that one
    for octaves in (18, 20, 21, 22, 23, 26, 29, 32, 34, 36):
        w = torch.zeros(c.pages, 1, 256, device="cuda") if accounts else None
        _, out = c.attend([news], heads, dtype, q=q, scale=octaves * np.log(2.0) / dim, accounts=w)
        share = others * 2.0 ** -octaves
        want = (share / (1 + share))[:, None, None]
        bound = n * 2.0 ** (-31 if dtype == "bf16" else -34 if dim == 256 else -37) + want * (n * EPS + octaves * 2.0 ** -21 + (2.0 ** -8 + 2.0 ** -11 if dtype == "bf16" else 2.0 ** -21))
        assert np.all(np.abs(out - want) <= bound), (octaves, np.abs(out - want).max(), bound.max())


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("dim", (64, 128, 256))
@pytest.mark.parametrize("news", (1, 40))
def test_a_scale_of_nan(gpu, dtype, dim, news):
    """Rows that see a token are NaN, whichever kernel they take."""
    c = Case(gpu, [90], 2, dim, 64, seed=dim).fill()
    _, out = c.attend([news], 4, dtype, scale=float("nan"))
    assert np.isnan(out).all()


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
def test_tiny_keys_and_values_are_exact_operands(gpu, dtype):
    """Values whose scales are fp16 denormals: the matrix instructions must not flush them."""
    c = Case(gpu, [100], 1, 64, 32, seed=5)
    c.k = [x * np.float32(2e-6) for x in c.k]
    c.v = [x * np.float32(2e-6) for x in c.v]
    c.fill()
    q = 1e6 * gpu.randn(1, 2, 64, device="cuda")
    out = c.check([1], 2, dtype, q=q)
    assert np.abs(out).max() > 1e-8
    c.check([64], 2, dtype, q=1e6 * gpu.randn(64, 2, 64, device="cuda"))


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("news", (1, 64, 90))
def test_bad_tokens_reach_only_rows_that_see_them(gpu, dtype, news):
    """A NaN in a key or value makes the rows that attend to it NaN, and no other: not those in front of it, not those whose window has
    left it, not other heads; what lies behind a sequence in its pages reaches nobody."""
    c = Case(gpu, [150, 150], 2, 128, 64, seed=6)
    c.k[0][100, 0, 3] = np.nan
    c.v[0][120, 1, 3] = np.inf
    c.cache.random_(0, 256)  # (scales of every kind in the places that no token has)
    c.cache[:, :, :, 34 * 128:] = 0
    c.fill()
    for window in (0, 20):
        out = c.check([news, news], 4, dtype, window, with_accounts=True)
        assert np.isnan(out).any() == (news > 1 or window == 0) and not np.isnan(out).all()
    q = gpu.randn(2 * news, 4, 128, device="cuda")
    q[0, 1, 5] = float("nan")
    c.check([news, news], 4, dtype, q=q)


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
def test_rows_of_strange_layout(gpu, dtype):
    """Queries as a view of a wider projection, and at an offset and strides that no vector load fits: the same results."""
    torch = gpu
    c = Case(torch, [77, 200], 2, 64, 32, seed=7).fill()
    kind = {"f32": torch.float32, "bf16": torch.bfloat16}[dtype]
    starts = c.ints([0, 40, 43])
    q = torch.randn(43, 6, 64, device="cuda").to(kind)
    args = (c.cache, c.d_table, c.ints(c.lengths))
    want = c.nn.cached_attention(q, *args, starts=starts, max_new=40)
    wide = torch.zeros(43, 10, 64, device="cuda", dtype=kind)
    wide[:, 2:8] = q
    assert torch.equal(c.nn.cached_attention(wide[:, 2:8], *args, starts=starts, max_new=40), want)
    odd = torch.zeros(43 * 6 * 67 + 1, device="cuda", dtype=kind)[1:].as_strided((43, 6, 64), (6 * 67, 67, 1), 1)
    odd.copy_(q)
    assert torch.equal(c.nn.cached_attention(odd, *args, starts=starts, max_new=40), want)
    # a wider table, and a slice of one
    wider = torch.full((2, 50), 7, dtype=torch.int32, device="cuda")
    wider[:, :c.table.shape[1]] = c.d_table
    got = c.nn.cached_attention(q, c.cache, wider[:, :c.table.shape[1]], c.ints(c.lengths), starts=starts, max_new=40)
    assert torch.equal(got, want)
    got = c.nn.cached_attention(q, c.cache, wider, c.ints(c.lengths), starts=starts, max_new=43).double()
    assert (got - want.double()).abs().max() <= (2.0 ** -8 if dtype == "bf16" else 2.0 ** -18) * want.double().abs().max()


def test_device_values_that_lead_nowhere(gpu):
    """Lengths past the table, starts past the rows, pages that are none of the cache's: cut off or absent, never followed."""
    torch = gpu
    c = Case(torch, [100, 90], 2, 64, 32, seed=8, wide_table=1).fill()
    q = torch.randn(2, 4, 64, device="cuda")
    table = c.d_table.clone()
    table[0, 1], table[1, 0] = -5, 10 ** 9
    out = c.nn.cached_attention(q, c.cache, table, c.ints([100, 90]))
    host = c.host()
    for b, gone in ((0, range(32, 64)), (1, range(0, 32))):
        for h in range(2):
            keys, values = ref.decode(host, c.table[b], c.lengths[b], h)
            left = [t for t in range(c.lengths[b]) if t not in gone]
            want, p, s, seen = ref.attention(q[b:b + 1, 2 * h:2 * h + 2].double().cpu().numpy(), keys[left], values[left], 0.125, 0)
            bound, _ = attention_bound(q[b:b + 1, 2 * h:2 * h + 2].double().cpu().numpy(), keys[left], values[left], 0.125, p, s, seen, "f32")
            assert np.all(np.abs(out[b, 2 * h:2 * h + 2].double().cpu().numpy() - want[0]) <= bound[0] + np.abs(want[0]) * 2 * EPS)
    weights = torch.zeros(c.pages, 2, 32, device="cuda")
    for lengths, starts in (([10 ** 9, -7], [0, 1, 2]), ([100, 90], [-3, 10 ** 6, 2]), ([100, 90], [2, 1, 0])):
        c.nn.cached_attention(q, c.cache, c.d_table, c.ints(lengths), starts=c.ints(starts), max_new=2, weights=weights)
        c.nn.kv_cache_append(c.cache, q[:, :2], q[:, 2:], c.d_table, c.ints(lengths), starts=c.ints(starts), max_new=2, weights=weights)
        c.nn.kv_cache_read(c.cache, c.d_table, c.ints(lengths), starts=c.ints(starts), max_new=2, rows=2)
        c.nn.kv_cache_evict(c.cache, weights, c.d_table, c.ints(lengths), 50, 10)
    torch.cuda.synchronize()


def absent_case(torch, length, rows, heads, room, dim, seed):
    """Two sequences of `room` cached tokens, of which the first says that it has `length` with `rows` new ones; a plain copy of everything."""
    c = Case(torch, [room, room], 2, dim, 32, seed=seed).fill()
    accounts = torch.from_numpy(c.rng.random((c.pages, 2, 32)).astype(np.float32)).cuda()
    k, v, q = (torch.from_numpy(c.rng.standard_normal((rows, h, dim)).astype(np.float32)).cuda() for h in (2, 2, heads))
    return c, accounts, k, v, q


@pytest.mark.parametrize("dim", (64, 128, 256))
@pytest.mark.parametrize("length,rows,max_new", ((130, 4, 4), (150, 60, 60), (129, 1, 1), (300, 40, 40), (100, 10, 6), (100, 70, 30), (150, 70, 40), (50, 90, 60)))
def test_tokens_without_a_place(gpu, dim, length, rows, max_new):
    """A sequence that has outgrown its page table, and rows behind the first max_new: new tokens lie where the length says, those without a place are
    absent, and nothing else moves: not the cached tokens in front, their accounts, nor other pages."""
    torch, room, heads = gpu, 128, 4
    c, accounts, k, v, q = absent_case(torch, length, rows, heads, room, dim, length + rows)
    nn, place = c.nn, [length - rows + n for n in range(min(rows, max_new))]
    stored = [n for n, p in enumerate(place) if 0 <= p < room]
    lengths, starts = c.ints([length, room]), c.ints([0, rows, rows])
    before, w0 = c.host().copy(), accounts.cpu().numpy()
    nn.kv_cache_append(c.cache, k, v, c.d_table, lengths, starts=starts, max_new=max_new, weights=accounts)
    host, w1 = c.host(), accounts.cpu().numpy()
    new = ref.quantise(k.cpu().numpy(), v.cpu().numpy())
    expect = w0.copy()
    for n in stored:
        expect[c.table[0, place[n] // 32], :, place[n] % 32] = 0
    assert np.array_equal(w1, expect)
    for h in range(2):
        for i, (x, y) in enumerate(zip(ref.decode(before, c.table[0], room, h), ref.decode(host, c.table[0], room, h))):
            for n in stored:
                x[place[n]] = new[i][n, h]
            assert np.array_equal(x, y)
    others = sorted(set(range(c.pages)) - set(c.table[0].tolist()))
    assert np.array_equal(before[others], host[others])
    got = nn.kv_cache_read(c.cache, c.d_table, lengths, starts=starts, max_new=max_new, rows=rows)
    for i, x in enumerate(got):
        x = x.double().cpu().numpy()
        for n, p in enumerate(place):
            want = np.zeros((2, dim)) if not 0 <= p < room else np.stack([ref.decode(host, c.table[0], room, h)[i][p] for h in range(2)])
            assert np.array_equal(x[n], want)
    for dtype in ("f32", "bf16"):
        for window in (0, 45):
            w = torch.from_numpy(w0).cuda()
            qd = q.to({"f32": torch.float32, "bf16": torch.bfloat16}[dtype])
            out = nn.cached_attention(qd, c.cache, c.d_table, lengths, starts=starts, max_new=max_new, window=window, weights=w).double().cpu().numpy()
            total, slack = w0.astype(np.float64), np.abs(w0.astype(np.float64)) * 2 * EPS
            for h in range(2):
                keys, values = ref.decode(host, c.table[0], room, h)
                for n, p in enumerate(place):
                    lo, hi = max(0, p + 1 - window if window else 0), min(p + 1, room)
                    y = out[n, 2 * h:2 * h + 2]
                    if lo >= hi:
                        assert np.all(y == 0)
                        continue
                    x = qd[n:n + 1, 2 * h:2 * h + 2].double().cpu().numpy()
                    want, share, s, seen = ref.attention(x, keys[lo:hi], values[lo:hi], dim ** -0.5, 0)
                    bound, eps_p = attention_bound(x, keys[lo:hi], values[lo:hi], dim ** -0.5, share, s, seen, dtype)
                    assert np.all(np.abs(y - want[0]) <= bound[0] + np.abs(want[0]) * (2.0 ** -8 if dtype == "bf16" else 2 * EPS))
                    t = np.arange(lo, hi)
                    total[c.table[0, t // 32], h, t % 32] += share[0].sum(0)
                    slack[c.table[0, t // 32], h, t % 32] += (share[0] * (eps_p[0][:, None] + (2 * len(place) + 4) * EPS)).sum(0) + total[c.table[0, t // 32], h, t % 32] * EPS
            assert np.all(np.abs(w.cpu().numpy() - total) <= slack)
    kept, left = nn.kv_cache_evict(c.cache, accounts, c.d_table, lengths, 300, 20)  # a length beyond the table ends with it
    assert left.tolist() == [min(length, room), room] and kept[0, 0].tolist() == [t if t < min(length, room) else -1 for t in range(300)]


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("rows", (1, 3, 40))
def test_windows_of_sequences_past_the_page_table(gpu, dtype, rows):
    """A window wider than the table still ends where it ends for rows whose places lie behind it; one wider than anything sees all there is."""
    torch, room, heads, dim = gpu, 128, 4, 64
    c, accounts, _, _, q = absent_case(torch, 300, rows, heads, room, dim, rows)
    q = q.to({"f32": torch.float32, "bf16": torch.bfloat16}[dtype])
    host, lengths, starts = c.host(), c.ints([300, room]), c.ints([0, rows, rows])
    for window in (128, 200, 255, 290, 400, 2 ** 31 - 1, 2 ** 40):
        w = torch.zeros_like(accounts)
        out = c.nn.cached_attention(q, c.cache, c.d_table, lengths, starts=starts, max_new=rows, window=window, weights=w).double().cpu().numpy()
        total = np.zeros(accounts.shape)
        for h in range(2):
            keys, values = ref.decode(host, c.table[0], room, h)
            for n in range(rows):
                lo = max(0, 300 - rows + n + 1 - window)
                y = out[n, 2 * h:2 * h + 2]
                if lo >= room:
                    assert np.all(y == 0)
                    continue
                x = q[n:n + 1, 2 * h:2 * h + 2].double().cpu().numpy()
                want, share, s, seen = ref.attention(x, keys[lo:], values[lo:], dim ** -0.5, 0)
                bound, _ = attention_bound(x, keys[lo:], values[lo:], dim ** -0.5, share, s, seen, dtype)
                assert np.all(np.abs(y - want[0]) <= bound[0] + np.abs(want[0]) * (2.0 ** -8 if dtype == "bf16" else 2 * EPS)), window
                t = np.arange(lo, room)
                total[c.table[0, t // 32], h, t % 32] += share[0].sum(0)
        assert np.all(np.abs(w.cpu().numpy() - total) <= 1e-4 * total)


@pytest.mark.parametrize("dim", (64, 128))
def test_single_tokens_past_the_page_table(gpu, dim):
    """Steps of one token each that go on past the table's end leave the cache alone, and attend to what there is."""
    torch = gpu
    c = Case(torch, [64, 40], 2, dim, 32, seed=dim).fill()
    before = c.host().copy()
    w = torch.ones(c.pages, 2, 32, device="cuda")
    q = torch.randn(2, 4, dim, device="cuda")
    want = c.nn.cached_attention(q, c.cache, c.d_table, c.ints([64, 40]))
    for step in range(1, 4):
        lengths = c.ints([64 + step, 40])
        c.nn.kv_cache_append(c.cache, q[:, :2], q[:, 2:], c.d_table, lengths, weights=w)
        c.lengths = [64, 40]
        host = c.host()
        for h in range(2):
            for x, y in zip(ref.decode(before, c.table[0], 64, h), ref.decode(host, c.table[0], 64, h)):
                assert np.array_equal(x, y)
        assert torch.equal(c.nn.cached_attention(q, c.cache, c.d_table, lengths)[0], want[0])
    gone = sorted(set(range(c.pages)) - set(c.table[1].tolist()))
    assert np.array_equal(host[gone], before[gone]) and np.all(w.cpu().numpy()[gone] == 1)


@pytest.mark.parametrize("dtype", ("f32", "bf16"))
def test_more_rows_than_a_launch_has_threads_for_one_by_one(gpu, dtype):
    """131072 new tokens of 128 heads, 2^24 rows, in one call: every one of them over its window."""
    torch = gpu
    from gomlx_amd import nn
    n, heads, dim, window = 131072, 128, 64, 64
    kind = {"f32": torch.float32, "bf16": torch.bfloat16}[dtype]
    gen = torch.Generator("cuda").manual_seed(3)
    k, v = (torch.randn(n, 1, dim, device="cuda", dtype=torch.bfloat16, generator=gen) for _ in range(2))
    table = torch.arange(n // 256, dtype=torch.int32, device="cuda").view(1, -1)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = nn.kv_cache(n // 256, 1, dim, 256)
    nn.kv_cache_append(cache, k, v, table, ints(n), starts=ints(0, n), max_new=n)
    q = torch.randn(1, heads, dim, device="cuda", generator=gen).to(kind)
    out = nn.cached_attention(q.expand(n, heads, dim), cache, table, ints(n), starts=ints(0, n), max_new=n, window=window)
    keys, values = (x[:, 0].double().cpu().numpy() for x in nn.kv_cache_read(cache, table, ints(n), starts=ints(0, n), max_new=n, rows=n))
    x = q.double().cpu().numpy()
    for p in [0, 1, 62, 63, 64, 65, 4095, 65535, 65536, 99999, 131008, 131071] + list(range(500, n, 9973)):
        lo = max(0, p + 1 - window)
        want, share, scores, seen = ref.attention(x, keys[lo:p + 1], values[lo:p + 1], dim ** -0.5, 0)
        bound, _ = attention_bound(x, keys[lo:p + 1], values[lo:p + 1], dim ** -0.5, share, scores, seen, dtype)
        assert np.all(np.abs(out[p].double().cpu().numpy() - want[0]) <= bound[0] + np.abs(want[0]) * (2.0 ** -8 if dtype == "bf16" else 2 * EPS)), p


@pytest.mark.parametrize("news", (1, 40))
def test_a_page_table_wider_than_a_launch(gpu, news):
    """A table with room for 2^29 tokens: attention goes by the tokens that there are; accounts, whose workgroups are laid out by its width, ask for a slice of it
    where they are too many."""
    torch = gpu
    from gomlx_amd import _lib
    c = Case(torch, [100], 2, 64, 64, seed=news).fill()
    wide = torch.full((1, 1 << 23), -1, dtype=torch.int32, device="cuda")
    wide[:, :c.table.shape[1]] = c.d_table
    q = torch.randn(news, 4, 64, device="cuda")
    how = dict(starts=c.ints([0, news]), max_new=news)
    want, got = (c.nn.cached_attention(q, c.cache, t, c.ints([100]), **how).double() for t in (c.d_table, wide))
    assert (got - want).abs().max() <= 2.0 ** -18 * want.abs().max()
    weights = [torch.zeros(c.pages, 2, 64, device="cuda") for _ in range(2)]
    c.nn.cached_attention(q, c.cache, c.d_table, c.ints([100]), weights=weights[0], **how)
    if news == 1:  # (16 rows and fewer: four tiles a workgroup)
        c.nn.cached_attention(q, c.cache, wide, c.ints([100]), weights=weights[1], **how)
        assert (weights[0] - weights[1]).abs().max() <= 2.0 ** -18
    else:
        with pytest.raises(_lib.HipqError, match="first columns"):
            c.nn.cached_attention(q, c.cache, wide, c.ints([100]), weights=weights[1], **how)
        c.nn.cached_attention(q, c.cache, wide[:, :1 << 22], c.ints([100]), weights=weights[1], **how)
        assert (weights[0] - weights[1]).abs().max() <= 2.0 ** -18 * news


def test_cache_past_four_gigabytes(gpu):
    """Pages whose bytes lie beyond 2^32."""
    torch = gpu
    from gomlx_amd import nn
    pages = (9 << 29) // (8 * 8 * 36 * 256)  # 4.8 GB
    cache = nn.kv_cache(pages, 8, 256, 256)
    assert cache.numel() > 1 << 32
    table = torch.tensor([[pages - 1, 3]], dtype=torch.int32, device="cuda")
    small, t2 = nn.kv_cache(2, 8, 256, 256), torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    k, v, q = (torch.randn(300, 8, 256, device="cuda") for _ in range(3))
    n = torch.tensor([300], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 300], dtype=torch.int32, device="cuda")
    outs = []
    for c, t in ((cache, table), (small, t2)):
        w = torch.zeros(c.shape[0], 8, 256, device="cuda")
        nn.kv_cache_append(c, k, v, t, n, starts=starts, max_new=300)
        a = nn.cached_attention(q, c, t, n, starts=starts, max_new=300, weights=w)
        b = nn.cached_attention(q[:1], c, t, n)
        kept, left = nn.kv_cache_evict(c, w, t, n, 200, 20)
        outs.append((a, b, kept, *nn.kv_cache_read(c, t, left, starts=torch.tensor([0, 200], dtype=torch.int32, device="cuda"), max_new=200, rows=200)))
    for x, y in zip(*outs):
        assert torch.equal(x, y)


# ---- eviction ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dim,page", ((64, 32), (128, 64), (256, 96)))
@pytest.mark.parametrize("keep,recent", ((1, 0), (1, 1), (32, 7), (45, 45), (150, 0), (333, 40), (2000, 5)))
def test_evict(gpu, dim, page, keep, recent):
    """Places, order, codes, scales and accounts of what stays; sequences within the budget are left alone."""
    torch = gpu
    lengths = [0, 1, 32, 45, 150, 700, 1500]
    c = Case(torch, lengths, 2, dim, page, seed=keep).fill()
    accounts = np.round(c.rng.standard_normal((c.pages, 2, page)).astype(np.float32) ** 2, 1)  # many exactly equal
    accounts[c.rng.random(accounts.shape) < 0.3] = 0
    accounts[c.rng.random(accounts.shape) < 0.01] = np.nan
    accounts[c.rng.random(accounts.shape) < 0.01] = np.inf
    accounts[c.rng.random(accounts.shape) < 0.05] *= -1
    d = torch.from_numpy(accounts).cuda()
    before = c.host().copy()
    kept, left = c.nn.kv_cache_evict(c.cache, d, c.d_table, c.ints(lengths), keep, recent)
    kept, after, d = kept.cpu().numpy(), c.host(), d.cpu().numpy()
    assert left.tolist() == [min(n, keep) for n in lengths]
    for b, n in enumerate(lengths):
        where = [(c.table[b, t // page], t % page) for t in range(n)]
        for h in range(2):
            want = ref.evict(np.array([accounts[p, h, s] for p, s in where], np.float32), keep, recent)
            assert kept[b, h].tolist() == want.tolist() + [-1] * (keep - len(want))
            old, new = ref.decode(before, c.table[b], n, h), ref.decode(after, c.table[b], n, h)
            for i in (0, 1):
                assert np.array_equal(new[i][:len(want)], old[i][want])
                assert np.array_equal(new[i][len(want):], old[i][len(want):])  # what lies behind is left as it was
            got = np.array([d[p, h, s] for p, s in where], np.float32)
            assert np.array_equal(got[:len(want)], np.array([accounts[where[t][0], h, where[t][1]] for t in want], np.float32), equal_nan=True)


@pytest.mark.parametrize("length", (4096, 4097, 16500, 40000))
@pytest.mark.parametrize("kind", ("spread", "few", "same", "zeros", "signs", "crowded"))
def test_evict_long_sequences(gpu, length, kind):
    """The selection alone over lengths that take each of its forms, and accounts that are hard on it."""
    torch = gpu
    from gomlx_amd import nn
    rng = np.random.default_rng(length)
    accounts = {"spread": np.exp(8 * rng.standard_normal(length)), "few": rng.integers(0, 3, length), "same": np.full(length, 0.7),
                "zeros": np.where(rng.random(length) < 0.01, rng.random(length), 0), "crowded": 1 + 1e-4 * rng.random(length), "signs": 1e30 * rng.standard_normal(length)}[kind].astype(np.float32)
    if kind == "signs":
        accounts[::50], accounts[1::50], accounts[2::50] = -0.0, np.inf, -np.inf
    if kind == "crowded":  # thousands share every digit but the last
        accounts[::1000], accounts[7::1000] = 1e30, 1e-30
    pages = -(-length // 64)
    cache, table = nn.kv_cache(pages, 1, 64, 64), torch.randperm(pages, device="cuda").int().view(1, -1)
    w = torch.zeros(pages, 1, 64, device="cuda")
    padded = np.zeros(pages * 64, np.float32)
    padded[:length] = accounts
    w[table[0].long(), 0] = torch.from_numpy(padded).cuda().view(pages, 64)
    n = torch.tensor([length], dtype=torch.int32, device="cuda")
    for keep, recent in ((1, 0), (length // 3, 100), (length - 1, 0), (length // 2, length // 2)):
        kept, _ = nn.kv_cache_evict(cache, w.clone(), table, n, keep, recent)
        assert kept[0, 0].tolist() == ref.evict(accounts, keep, recent).tolist()


@pytest.mark.parametrize("choose", (4096, 16384, 16416, 32768, 32800))
def test_evict_at_the_ends_of_the_selections_forms(gpu, choose):
    """As many tokens to choose from as one form takes and the next: kept in registers, in LDS, or read again.  Ties among them."""
    torch = gpu
    from gomlx_amd import nn
    rng = np.random.default_rng(choose)
    length, recent = choose + 32, 32
    accounts = np.round(4 * rng.standard_normal((2, length))).astype(np.float32)
    pages = length // 32
    cache, table = nn.kv_cache(pages, 2, 64, 32), torch.arange(pages, device="cuda").int().view(1, -1)
    w = torch.from_numpy(accounts).cuda().view(2, pages, 32).transpose(0, 1).contiguous()
    n = torch.tensor([length], dtype=torch.int32, device="cuda")
    for keep in (recent + 1, length // 2, length - 1):
        kept, _ = nn.kv_cache_evict(cache, w.clone(), table, n, keep, recent)
        for h in range(2):
            assert kept[0, h].tolist() == ref.evict(accounts[h], keep, recent).tolist()


def test_every_scale(gpu):
    """The quotient that codes are rounded from, over every scale that there is and values around every code's border."""
    torch = gpu
    from gomlx_amd import nn
    bits = np.arange(1, 0x7C00, dtype=np.uint16).view(np.float16).astype(np.float32)
    scales = np.array([d for d in bits if d <= 8160 and ref._bf16(np.float32([d]))[0] == d], np.float32)
    k = np.zeros((len(scales), 1, 64), np.float32)
    for i, d in enumerate(scales):
        border = (np.arange(-8, 8, dtype=np.float64) + 0.5) * d
        near = np.concatenate([border, np.nextafter(border.astype(np.float32), np.float32(np.inf)), np.nextafter(border.astype(np.float32), np.float32(-np.inf)),
                               border * (1 + 1e-6 * np.random.default_rng(i).standard_normal(16))]).astype(np.float32)
        k[i, 0] = np.clip(near, -7.99 * d, 7.99 * d)
        k[i, 0, [5, 40]] = -8 * d, 8 * d
    cache = nn.kv_cache(-(-len(scales) // 256), 1, 64, 256)
    table = torch.arange(cache.shape[0], dtype=torch.int32, device="cuda").view(1, -1)
    n, starts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([len(scales)], [0, len(scales)]))
    d = torch.from_numpy(k).cuda()
    nn.kv_cache_append(cache, d, -d, table, n, starts=starts, max_new=len(scales))
    got = nn.kv_cache_read(cache, table, n, starts=starts, max_new=len(scales), rows=len(scales))
    for x, y in zip(got, ref.quantise(k, -k)):
        assert np.array_equal(x.double().cpu().numpy(), y)


def test_evict_writes_lengths_in_place_and_goes_on(gpu):
    """Serving: append, attend with accounts, evict into the same lengths, go on with the shorter sequences."""
    torch = gpu
    from gomlx_amd import _lib
    import ctypes
    c = Case(torch, [130, 60], 1, 64, 32, seed=2, wide_table=1).fill()
    weights = torch.zeros(c.pages, 1, 32, device="cuda")
    q = torch.randn(2, 4, 64, device="cuda")
    lengths = c.ints([130, 60])
    c.nn.cached_attention(q, c.cache, c.d_table, lengths, weights=weights)
    kept = torch.empty(2, 1, 64, dtype=torch.int32, device="cuda")
    d = c.nn._kv_desc(c.cache, c.d_table, lengths, accounts=weights)
    _lib.check(_lib.lib().gq_kv_evict(ctypes.byref(d), weights.data_ptr(), 64, 16, kept.data_ptr(), lengths.data_ptr(), torch.cuda.current_stream().cuda_stream))
    assert lengths.tolist() == [64, 60]
    k, v = (torch.randn(2, 1, 64, device="cuda") for _ in range(2))
    c.nn.kv_cache_append(c.cache, k, v, c.d_table, lengths + 1, weights=weights)
    c.lengths = [65, 61]
    c.check([1, 1], 4)


# ---- norms and rotation ---------------------------------------------------------------------------------------------------


def rope_bound(size, want, dtype):
    """The sum of squares is a sum of D positive terms in float32 (relative error up to D 2^-24 halved by the root), then a root, a
    division, two products and a sum: under (D / 2 + 8) 2^-24 of the two terms' magnitudes; bfloat16 results are rounded to 2^-8."""
    return size * (size.shape[-1] / 2 + 8) * EPS + (np.abs(want) * 2.0 ** -8 if dtype == "bf16" else 0)


@pytest.mark.parametrize("dim,rot", ((64, 64), (128, 128), (128, 64), (256, 256), (256, 8), (64, 24), (128, 0)))
@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("kind,out", (("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "f32")))
def test_qk_norm_rope(gpu, dim, rot, interleaved, kind, out):
    torch = gpu
    from gomlx_amd import nn
    rng = np.random.default_rng(dim + rot)
    types = {"f32": torch.float32, "bf16": torch.bfloat16}
    cos, sin = nn.rotary_table(5000, rot, 10000.0) if rot else (torch.zeros(5000, 0, device="cuda"),) * 2
    for rows, heads, kv, norm in ((1, 4, 1, True), (37, 6, 2, True), (5, 3, 3, False), (3, 0, 2, True), (0, 4, 2, True)):
        wide = torch.from_numpy(rng.standard_normal((rows, (heads + 2 * kv) * dim)).astype(np.float32)).cuda().to(types[kind])
        q, k = wide[:, :heads * dim].view(rows, heads, dim), wide[:, heads * dim:(heads + kv) * dim].view(rows, kv, dim)
        pos = rng.integers(0, 5000, rows).astype(np.int32)
        if rows > 4:
            pos[1], pos[3] = -1, 5000  # outside the table
        gains = [torch.from_numpy(rng.standard_normal(dim).astype(np.float32)).cuda(), None]
        norms = [nn.RMSNorm(gain=gains[0], epsilon=1e-5, scale_offset=1.0), nn.RMSNorm(epsilon=1e-6)] if norm else [None, None]
        got = nn.qk_norm_rope(q, k, torch.from_numpy(pos).cuda(), cos, sin, *norms, interleaved=interleaved, dtype=types[out])
        for x, y, g, n in zip((q, k), got, gains, norms):
            assert y.shape == x.shape and y.dtype == types[out] and y.is_contiguous()
            want, size = ref.norm_rope(x.double().cpu().numpy(), pos, cos.cpu().numpy(), sin.cpu().numpy(), None if g is None else g.cpu().numpy(),
                                       n.epsilon if n else 0.0, n.scale_offset if n else 0.0, norm, interleaved)
            y = y.double().cpu().numpy()
            assert np.array_equal(np.isnan(y), np.isnan(want))
            fine = ~np.isnan(want)
            assert np.all(np.abs(y - want)[fine] <= rope_bound(size, want, out)[fine])


def test_qk_norm_rope_rows_off_every_vector(gpu):
    torch = gpu
    from gomlx_amd import nn
    cos, sin = nn.rotary_table(64, 128)
    pos = torch.arange(9, dtype=torch.int32, device="cuda")
    for kind in (torch.float32, torch.bfloat16):
        q, k = (torch.randn(9, 2, 128, device="cuda").to(kind) for _ in range(2))
        odd = [torch.zeros(9 * 2 * 131 + 1, dtype=kind, device="cuda")[1:].as_strided((9, 2, 128), (2 * 131, 131, 1), 1) for _ in range(2)]
        for o, x in zip(odd, (q, k)):
            o.copy_(x)
        for a, b in zip(nn.qk_norm_rope(q, k, pos, cos, sin), nn.qk_norm_rope(*odd, pos, cos, sin)):
            assert torch.equal(a, b)
    zero = torch.zeros(9, 2, 128, device="cuda")
    a, _ = nn.qk_norm_rope(zero, zero, pos, cos, sin, q_norm=nn.RMSNorm())  # eps keeps a head of zeros at zero
    assert torch.equal(a, zero)


@pytest.mark.parametrize("dim", (64, 128, 256))
@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("kind", ("f32", "bf16"))
def test_qk_norm_rope_without_a_table(gpu, dim, interleaved, kind):
    """A table of no rows, which has no memory, and one cut to no rows: every position lies outside, every row is NaN."""
    torch = gpu
    from gomlx_amd import nn
    q, k = (torch.randn(5, h, dim, device="cuda").to({"f32": torch.float32, "bf16": torch.bfloat16}[kind]) for h in (3, 1))
    pos = torch.tensor([0, 1, -1, 7, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    full = nn.rotary_table(8, dim)
    for cos, sin in (nn.rotary_table(0, dim), [t[:0] for t in full], nn.rotary_table(0, 8)):
        for y in nn.qk_norm_rope(q, k, pos, cos, sin, q_norm=nn.RMSNorm(), interleaved=interleaved):
            assert y.isnan().all()
    for y in nn.qk_norm_rope(q, k, pos, *full, interleaved=interleaved):
        assert y.isnan().all(-1).all(-1).tolist() == [False, False, True, False, True] and y.isnan().any(-1).any(-1).tolist() == [False, False, True, False, True]


def test_qk_norm_rope_of_more_heads_than_a_launch_has_threads_for(gpu):
    """2^26 and some heads of 256 values, one head over and over (34 GB of results)."""
    torch = gpu
    from gomlx_amd import nn
    rows, heads, dim = (1 << 20) + 3, 64, 256
    one = torch.randn(1, heads, dim, device="cuda", dtype=torch.bfloat16)
    cos, sin = nn.rotary_table(16, dim)
    pos = (torch.arange(rows, device="cuda") % 16).int()
    q, k = nn.qk_norm_rope(one.expand(rows, heads, dim), one[:, :0].expand(rows, 0, dim), pos, cos, sin)
    want, _ = nn.qk_norm_rope(one.expand(1024, heads, dim), one[:, :0].expand(1024, 0, dim), pos[:1024].contiguous(), cos, sin)
    assert k.shape == (rows, 0, dim)
    for at in range(0, rows, 1024):
        n = min(1024, rows - at)
        assert torch.equal(q[at:at + n], want[:n]), at
    del q
    torch.cuda.empty_cache()


# ---- together -----------------------------------------------------------------------------------------------------------


def test_recorded_graph_replays_over_growing_sequences(gpu):
    """rotate, append, attend with accounts as one HIP graph, replayed while lengths and inputs change, with eager work between."""
    torch = gpu
    from gomlx_amd import nn
    dim, kv, heads, page, seqs = 64, 2, 4, 32, 3
    table = torch.arange(seqs * 6, dtype=torch.int32, device="cuda").view(seqs, 6)
    cos, sin = nn.rotary_table(256, dim)

    def state():
        return dict(cache=nn.kv_cache(seqs * 6, kv, dim, page), weights=torch.zeros(seqs * 6, kv, page, device="cuda"),
                    lengths=torch.tensor([90, 31, 1], dtype=torch.int32, device="cuda"), x=torch.zeros(seqs, heads + 2 * kv, dim, device="cuda"))

    def step(s):
        q, k = nn.qk_norm_rope(s["x"][:, :heads], s["x"][:, heads:heads + kv], s["lengths"], cos, sin, q_norm=nn.RMSNorm(), k_norm=nn.RMSNorm())
        nn.kv_cache_append(s["cache"], k, s["x"][:, heads + kv:], table, s["lengths"], weights=s["weights"])
        return nn.cached_attention(q, s["cache"], table, s["lengths"], weights=s["weights"])

    a, b = state(), state()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(b)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step(b)
    for s in (a, b):
        s["cache"].zero_()
        s["weights"].zero_()
    for i in range(5):
        x = torch.randn(seqs, heads + 2 * kv, dim, device="cuda")
        for s in (a, b):
            s["x"].copy_(x)
            s["lengths"] += 1
        want = step(a)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(a["cache"], b["cache"]) and torch.equal(a["weights"], b["weights"])


def test_two_streams(gpu):
    """Calls on two streams have workspaces of their own."""
    torch = gpu
    c = Case(torch, [3000], 2, 128, 64, seed=11).fill()
    qs = [torch.randn(1, 8, 128, device="cuda") for _ in range(2)]
    n = c.ints([3000])
    want = [c.nn.cached_attention(q, c.cache, c.d_table, n) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(20):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                outs[i].append(c.nn.cached_attention(qs[i], c.cache, c.d_table, n))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(o, want[i]) for o in outs[i])


def test_same_call_same_bits(gpu):
    torch = gpu
    c = Case(torch, [700, 650], 2, 128, 64, seed=12).fill()
    q = torch.randn(100, 8, 128, device="cuda")
    starts = c.ints([0, 60, 100])
    runs = []
    for _ in range(3):
        w = torch.zeros(c.pages, 2, 64, device="cuda")
        runs.append((c.nn.cached_attention(q, c.cache, c.d_table, c.ints(c.lengths), starts=starts, max_new=60, weights=w), w))
    for o, w in runs[1:]:
        assert torch.equal(o, runs[0][0]) and torch.equal(w, runs[0][1])


def test_refusals(gpu):
    torch = gpu
    from gomlx_amd import _lib, nn
    c = Case(torch, [40, 10], 2, 64, 32).fill()
    n = c.ints([40, 10])
    q = torch.zeros(2, 4, 64, device="cuda")
    k = torch.zeros(2, 2, 64, device="cuda")
    w = torch.zeros(c.pages, 2, 32, device="cuda")
    good = dict(q=q, cache=c.cache, page_table=c.d_table, lengths=n)
    for change, error in ((dict(q=q.half()), _lib.NotImplementedByBackend), (dict(q=q[:, :3]), ValueError), (dict(q=q[:1]), ValueError), (dict(q=q[..., ::2]), ValueError),
                          (dict(q=q.cpu()), ValueError), (dict(q=q.view(2, 256)), ValueError), (dict(cache=c.cache[..., :-36]), ValueError),
                          (dict(cache=c.cache.view(torch.int8)), ValueError), (dict(lengths=n.long()), ValueError), (dict(page_table=c.d_table[:1]), ValueError),
                          (dict(page_table=c.d_table.long()), ValueError), (dict(window=-1), ValueError), (dict(starts=c.ints([0, 2])), ValueError),
                          (dict(max_new=2), ValueError), (dict(starts=c.ints([0, 1, 2]), max_new=0), ValueError), (dict(weights=w[:, :1]), ValueError),
                          (dict(weights=w.double()), ValueError)):
        with pytest.raises(error):
            nn.cached_attention(**{**good, **change})
    with pytest.raises(ValueError):
        nn.kv_cache_append(c.cache, k, k.bfloat16(), c.d_table, n)
    with pytest.raises(ValueError):
        nn.kv_cache_append(c.cache, k[:, :1], k[:, :1], c.d_table, n)
    with pytest.raises(_lib.NotImplementedByBackend):
        nn.kv_cache_append(c.cache, k.half(), k.half(), c.d_table, n)
    with pytest.raises(ValueError):
        nn.kv_cache_read(c.cache, c.d_table, n, starts=c.ints([0, 1, 2]), max_new=1)
    for keep, recent in ((0, 0), (5, 6), (5, -1)):
        with pytest.raises(ValueError):
            nn.kv_cache_evict(c.cache, w, c.d_table, n, keep, recent)
    with pytest.raises(ValueError):
        nn.kv_cache_evict(c.cache, None, c.d_table, n, 5, 1)
    cos, sin = nn.rotary_table(10, 64)
    pos = c.ints([0, 1])
    good = dict(q=q, k=k, positions=pos, cos=cos, sin=sin)
    for change, error in ((dict(q=q.half(), k=k.half()), _lib.NotImplementedByBackend), (dict(k=k.bfloat16()), ValueError), (dict(k=k[:1]), ValueError),
                          (dict(q=q[..., :32].contiguous(), k=k[..., :32].contiguous()), _lib.NotImplementedByBackend), (dict(positions=pos.long()), ValueError),
                          (dict(sin=sin[:5]), ValueError), (dict(cos=cos[:, :30].contiguous(), sin=sin[:, :30].contiguous()), _lib.HipqError),
                          (dict(cos=cos.double(), sin=sin.double()), ValueError), (dict(dtype=torch.float16), _lib.NotImplementedByBackend),
                          (dict(q_norm=nn.RMSNorm(gain=torch.ones(32, device="cuda"))), ValueError)):
        with pytest.raises(error):
            nn.qk_norm_rope(**{**good, **change})
    for bad in (dict(head_dim=80), dict(page_tokens=33), dict(kv_heads=0)):
        with pytest.raises((ValueError, _lib.NotImplementedByBackend)):
            nn.kv_cache(**{**dict(pages=1, kv_heads=1, head_dim=64, page_tokens=32), **bad})


def test_native_host_path(gpu, monkeypatch):
    """The native steps serve the calls of a decode loop, with the Python steps' results; what they do not know they leave alone."""
    torch = gpu
    from gomlx_amd import _lib, nn
    c = Case(torch, [90, 33], 2, 64, 32, seed=1, wide_table=1).fill()
    n, starts = c.ints([90, 33]), c.ints([0, 4, 6])
    cos, sin = nn.rotary_table(100, 64)
    x = torch.randn(2, 10, 64, device="cuda")
    many = torch.randn(6, 4, 64, device="cuda").bfloat16()
    gain = nn.RMSNorm(gain=torch.randn(64, device="cuda"), epsilon=1e-5, scale_offset=1.0)
    fast = _lib.fast
    assert fast is not None

    def calls():
        w = torch.zeros(c.pages, 2, 32, device="cuda")
        cache = c.cache.clone()
        q, k = nn.qk_norm_rope(x[:, :4], x[:, 4:6], n, cos, sin, gain, nn.RMSNorm(), True, torch.bfloat16)
        out = [q, k, *nn.qk_norm_rope(x[:, :4], x[:, 4:6], n, cos, sin)]
        out.append(nn.kv_cache_append(cache, k, x[:, 6:8].bfloat16(), c.d_table, n + 1, weights=w))
        out.append(nn.kv_cache_append(cache, many[:, :2], many[:, 2:], c.d_table, n, starts=starts, max_new=4))
        out += [cache.clone(), nn.cached_attention(q, cache, c.d_table, n + 1, weights=w), nn.cached_attention(many, cache, c.d_table, n, starts=starts, max_new=4, scale=0.3, window=9)]
        out += [*nn.kv_cache_read(cache, c.d_table, n), *nn.kv_cache_read(cache, c.d_table, n, starts, 4, 6), *nn.kv_cache_evict(cache, w, c.d_table, n, 40, 3), w, cache]
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
    assert all(ok for _, ok in served) and {name for name, _ in served} == {"qk_norm_rope", "kv_append", "kv_read", "cached_attention", "kv_evict"}
    monkeypatch.setattr(_lib, "fast", None)
    plain = calls()
    for a, b, d in zip(native, plain, spied):
        assert (a is None and b is None and d is None) or (torch.equal(a, b) and torch.equal(a, d) and a.dtype == b.dtype and a.stride() == b.stride())
    w = torch.zeros(c.pages, 2, 32, device="cuda")
    q = x[:, :4]
    for f, args in ((fast.cached_attention, (q.half(), c.cache, c.d_table, n, None, 1, None, 0, None)), (fast.cached_attention, (q[:, :3], c.cache, c.d_table, n, None, 1, None, 0, None)),
                    (fast.cached_attention, (q, c.cache, c.d_table, n, None, 2, None, 0, None)), (fast.cached_attention, (q, c.cache, c.d_table.long(), n, None, 1, None, 0, None)),
                    (fast.cached_attention, (q, c.cache, c.d_table, n, None, 1, None, -1, None)), (fast.cached_attention, (q, c.cache, c.d_table, n, None, 1, None, 0, w[:1])),
                    (fast.cached_attention, (q.cpu(), c.cache, c.d_table, n, None, 1, None, 0, None)), (fast.kv_append, (c.cache, q[:, :2], q[:, :2].bfloat16(), c.d_table, n, None, 1, None)),
                    (fast.kv_append, (c.cache, q[:1, :2], q[:1, :2], c.d_table, n, None, 1, None)), (fast.kv_read, (c.cache, c.d_table, n, starts, 4, None)),
                    (fast.kv_evict, (c.cache, None, c.d_table, n, 4, 0)), (fast.kv_evict, (c.cache, w, c.d_table, n, 4, 5)),
                    (fast.qk_norm_rope, (q, q[:1], n, cos, sin, None, None, False, None)), (fast.qk_norm_rope, (q, q, n, cos, sin[:3], None, None, False, None)),
                    (fast.qk_norm_rope, (q, q, n, cos, sin, None, None, False, torch.float16)), (fast.qk_norm_rope, (q, q, n.long(), cos, sin, None, None, False, None))):
        assert f(*args) is None


def test_empty_calls(gpu):
    torch = gpu
    from gomlx_amd import nn
    cache = nn.kv_cache(0, 2, 64, 32)
    table, n = torch.zeros(0, 3, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    q = torch.zeros(0, 4, 64, device="cuda")
    assert nn.cached_attention(q, cache, table, n).shape == (0, 4, 64)
    nn.kv_cache_append(cache, q[:, :2], q[:, :2], table, n)
    assert nn.kv_cache_read(cache, table, n)[0].shape == (0, 2, 64)
    kept, left = nn.kv_cache_evict(cache, torch.zeros(0, 2, 32, device="cuda"), table, n, 4)
    assert kept.shape == (0, 2, 4) and left.shape == (0,)
    # one sequence without a page: nothing to see
    cache, q = nn.kv_cache(1, 2, 64, 32), torch.randn(1, 4, 64, device="cuda")
    table, n = torch.zeros(1, 0, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    assert torch.equal(nn.cached_attention(q, cache, table, n, weights=torch.zeros(1, 2, 32, device="cuda")), torch.zeros_like(q))
    nn.kv_cache_append(cache, q[:, :2], q[:, 2:], table, n + 1)
    assert not cache.any()
