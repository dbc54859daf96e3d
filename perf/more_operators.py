"""Decoding with drafted tokens over a 4-bit cache, as cases to be timed: a step takes a tree of drafted tokens of every sequence through
the model at once and keeps the path that the model's own samples follow.

Four operators, in the order in which such a step calls them:

* tree    ``draft_tree``: from every row's parent the rows it sees, as bits, and its position;
* attend  ``tree_attention``: softmax attention of the drafted tokens, each over the cache in front of the tree and its own ancestors;
* sample  ``sample``: a token for every row of logits, from its temperature, top-k, top-p and min-p and a given random number;
* accept  ``kv_cache_accept``: the path of drafted tokens that the samples follow; their keys and values move behind one another in
          the cache (``kv_cache_read`` gives back what it then stands for), what was not accepted is left behind its new end.

With ``own`` false, ``run`` computes them from elementary torch operations; with ``own`` true it calls gomlx_amd.nn.

The cache, uint8 [pages, key heads, tiles of a page, 36 D]: a tile holds 32 tokens of one key head.  A group is 32 neighbouring
values of a head vector; it stands for d (c - 8) with a scale d (float16 of 8 significant bits) and codes c of 4 bits.

    bytes 0 to 16 D       key codes, dwords [w >> 2][lane][w & 3]: w = u D/32 + g, lane = 16 j + r;
                          token 8 (r >> 2) + 4 u + (r & 3), values 32 g + 8 j + e, e = 0 to 7
    bytes 16 D to 32 D    value codes, dwords [w >> 2][lane][w & 3]: lane = 16 j + r; tokens 8 j + e, value 16 w + r
                          (element e of a dword lies in its nibble (e >> 1) + 4 (e & 1))
    bytes 32 D to 34 D    key scales [token][group]
    bytes 34 D to 36 D    value scales [group][token]

Token p of sequence b lies in page ``page_table[b, p // tokens of a page]``.  ``lengths`` counts the tokens of a sequence with the drafted
ones; rows ``starts[b]`` to ``starts[b + 1]`` of a call's arguments are sequence b's drafted tokens, the last ones of it.  The first of
them is the tree's root, the token that the last step sampled; ``parents`` are rows counted from it, -1 for the root's.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    layer = dict(heads=32, kv_heads=8, dim=128)  # 4096 values as queries, 1024 as keys and as values
    small = dict(heads=12, kv_heads=12, dim=64)
    return [
        # The draft of one sequence: the smallest call, where latency counts.
        dict(name="tree_seq1", op="tree", seqs=1, nodes=8, depth=4),
        # The drafts of a large batch, of unlike sizes.
        dict(name="tree_seqs256", op="tree", seqs=256, nodes=64, depth=8),
        # One sequence in float32: few workgroups' worth of cache.
        dict(name="attend_seq1", op="attend", dtype="f32", seqs=1, nodes=8, depth=4, length=2047, page=64, window=0, **layer),
        # A decode batch in bfloat16 over caches of mixed lengths, sixteen drafted tokens for the longest.
        dict(name="attend_seqs32", op="attend", dtype="bf16", seqs=32, nodes=16, depth=5, length=8192, page=64, window=0, **layer),
        # A draft over one very long cache: the work is split along it and joined.
        dict(name="attend_long", op="attend", dtype="bf16", seqs=1, nodes=32, depth=6, length=131072, page=256, window=0, **layer),
        # Wide trees of a smaller batch: matrix products bound it.
        dict(name="attend_wide", op="attend", dtype="bf16", seqs=16, nodes=64, depth=8, length=8192, page=128, window=0, **layer),
        # Ragged trees in float32 with a window, smaller heads, one key head a query head.
        dict(name="attend_ragged", op="attend", dtype="f32", seqs=5, nodes=33, depth=7, length=1111, page=32, window=500, **small),
        # The next token of one sequence from a 128k-vocabulary output head.
        dict(name="sample_row1", op="sample", dtype="f32", rows=1, vocab=128256, temperature=0.8, top_k=50, top_p=0.9, min_p=0.0),
        # Every node of a batch's trees, each sequence with settings of its own.
        dict(name="sample_rows512", op="sample", dtype="f32", rows=512, vocab=128256, temperature=-1.0, top_k=-1, top_p=-1.0, min_p=-1.0),
        # bfloat16 logits of an odd vocabulary, many of them equal, by top-p alone.
        dict(name="sample_odd", op="sample", dtype="bf16", rows=33, vocab=50257, temperature=1.0, top_k=0, top_p=0.95, min_p=0.0),
        # The end of one sequence's step.
        dict(name="accept_seq1", op="accept", seqs=1, nodes=16, depth=5, length=2047, page=64, **layer),
        # The end of a large batch's step.
        dict(name="accept_seqs64", op="accept", seqs=64, nodes=64, depth=8, length=4096, page=128, **layer),
    ]


_MAX_FLOPS = 7.1e10   # of the largest listed cases (the wide trees)
_MAX_BYTES = 2.63e8   # the logits of 512 rows


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges."""
    while True:
        op = rng.choice(("tree", "attend", "attend", "attend", "attend", "sample", "sample", "sample", "accept"))
        if op == "sample":
            c = dict(op=op, dtype=rng.choice(("f32", "f32", "bf16")), rows=_log(rng, 1, 1024), vocab=_log(rng, 500, 262144))
            if rng.random() < 0.3:
                c.update(temperature=-1.0, top_k=-1, top_p=-1.0, min_p=-1.0)
            else:
                c.update(temperature=rng.choice((0.0, 0.6, 0.8, 1.0, 1.0, 1.3)), top_k=rng.choice((0, 0, 0, 1, 20, 50, _log(rng, 2, 2000))),
                         top_p=rng.choice((1.0, 1.0, 0.8, 0.9, 0.95, round(rng.uniform(0.05, 0.999), 3))), min_p=rng.choice((0.0, 0.0, 0.02, 0.1)))
        else:
            kv = rng.choice((1, 2, 4, 8, 8, 12, 16))
            c = dict(op=op, seqs=_log(rng, 1, 256 if op == "tree" else 48), nodes=_log(rng, 2, 96), depth=rng.randint(1, 10))
            if op != "tree":
                c.update(heads=kv * rng.choice((1, 2, 3, 4, 4, 7, 8)), kv_heads=kv, dim=rng.choice((64, 128, 128, 256)), page=rng.choice((32, 64, 96, 128, 256)),
                         length=c["nodes"] + _log(rng, 1, 30000))
            if op == "attend":
                c.update(dtype=rng.choice(("f32", "bf16", "bf16")), window=_log(rng, 16, c["length"]) if rng.random() < 0.25 else 0)
        w = work(c)
        # (the plain form holds keys and values in float32 and every score)
        cells = c.get("seqs", 0) * c.get("length", 0) * c.get("kv_heads", 0) * c.get("dim", 0)
        scores = c["seqs"] * c["length"] * c["heads"] * c["nodes"] if op == "attend" else 0
        if w["flops"] <= _MAX_FLOPS and w["bytes"] <= _MAX_BYTES and cells <= 3.0e8 and scores <= 3.0e8:
            return c


def _news(c):
    """Drafted tokens of each sequence: the most first, odd steps down to half of it."""
    return [max(1, c["nodes"] - b * c["nodes"] // (2 * c["seqs"])) for b in range(c["seqs"])]


def _lengths(c):
    """Tokens of each sequence with the drafted ones: the longest first, down to a quarter of it."""
    return [max(n, c["length"] - 3 * b * c["length"] // (4 * c["seqs"])) for b, n in enumerate(_news(c))]


def work(case):
    c = case
    if c["op"] == "tree":
        rows = sum(_news(c))
        return {"bytes": float(rows * (8 + 4 * -(-c["nodes"] // 32))), "flops": float(rows * c["depth"])}
    if c["op"] == "sample":
        return {"bytes": float(c["rows"] * c["vocab"] * (4 if c["dtype"] == "f32" else 2)), "flops": 4.0 * c["rows"] * c["vocab"]}
    D, rows = c["dim"], sum(_news(c))
    token = 36 * D // 32 * c["kv_heads"]  # bytes of a cached token
    if c["op"] == "accept":  # the accepted tokens read and written, and read back
        path = c["seqs"] * min(c["depth"] + 1, c["nodes"])
        return {"bytes": float(12 * rows + 3 * path * token + 4 * path * c["kv_heads"] * D), "flops": float(rows)}
    pairs = tokens = 0
    for n, length in zip(_news(c), _lengths(c)):
        seen = min(length - n + min(n, c["depth"] + 1), c["window"] or length)
        pairs += n * seen
        tokens += min(length, seen + n)
    return {"bytes": float(tokens * token + 2 * rows * c["heads"] * D * (4 if c["dtype"] == "f32" else 2)), "flops": 4.0 * D * c["heads"] * pairs}


# ---- the inputs ------------------------------------------------------------------------------------------------------


def _trees(c, seed):
    """Parents and tokens of every drafted row, and what the model samples there, as lists: levels of about equal size, the likeliest
    nodes of a level with the most children; a sample is a child's token three times out of four where there is one."""
    gen = torch.Generator()
    gen.manual_seed(seed)
    parents, tokens, sampled = [], [], []
    for n in _news(c):
        depth = min(c["depth"], n - 1)
        bounds = [0, 1] + [1 + (n - 1) * (i + 1) // depth for i in range(depth)] if depth else [0, 1]
        u = torch.rand(4, n, generator=gen, dtype=torch.float64)
        up, children = [-1], [[] for _ in range(n)]
        for lo, mid, hi in zip(bounds, bounds[1:], bounds[2:]):
            for i in range(mid, hi):
                up.append(lo + int((mid - lo) * float(u[0, i]) ** 2))
                children[up[i]].append(i)
        words = (32000 * u[1]).long().tolist()
        follows = []
        for i in range(n):
            some = children[i][int(len(children[i]) * float(u[3, i]) ** 2)] if children[i] and float(u[2, i]) < 0.75 else None
            follows.append(int(32000 * float(u[3, i])) if some is None else words[some])
        parents += up
        tokens += words
        sampled += follows
    return parents, tokens, sampled


def _bits(parents, counts, words):
    """What ``draft_tree`` makes of parents, row by row: [rows, words] of int32 as lists, and depths."""
    rows, depths, at = [], [], 0
    for n in counts:
        seen = []
        for i in range(n):
            p = parents[at + i]
            seen.append((seen[p] if p >= 0 else 0) | 1 << i)
            depths.append(depths[at + p] + 1 if p >= 0 else 0)
        for s in seen:
            w = [s >> (32 * j) & 0xFFFFFFFF for j in range(words)]
            rows.append([x - (1 << 32) if x >= 1 << 31 else x for x in w])
        at += n
    return rows, depths


def prepare(case, seed):
    c = dict(case)
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device=dev, generator=gen)

    def uniform(*shape):
        return torch.rand(shape, device=dev, generator=gen)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    if c["op"] == "sample":
        # logits as an output head leaves them: most of a vocabulary about alike, and a few tokens that fall off with their rank from
        # a height that says how sure the model is; of every eighth row it is not sure of much
        rows, vocab = c["rows"], c["vocab"]
        head = min(256, vocab)
        x = 1.5 * normal(rows, vocab)
        top = 14.0 + 9.0 * uniform(rows, 1)
        top[::8] = 10.0
        high = top - 1.5 * torch.arange(1, head + 1, device=dev).log() + 0.5 * normal(rows, head)
        # (where they are: as in vocabularies sorted by frequency more often at low indices)
        x.scatter_reduce_(1, (vocab * uniform(rows, head).double().square()).long(), high, "amax")
        st = dict(case=c, logits=x.to(DTYPES[c["dtype"]]), uniform=uniform(rows))
        if c["temperature"] < 0:  # settings of each row
            def choose(values, dtype):
                return torch.tensor(values, dtype=dtype, device=dev)[(len(values) * uniform(rows)).long()]
            st["settings"] = dict(temperature=choose([0.0, 0.6, 0.8, 1.0, 1.0, 1.2], torch.float32), top_k=choose([0, 0, 20, 50, 200], torch.int32),
                                  top_p=choose([1.0, 0.8, 0.9, 0.95], torch.float32), min_p=choose([0.0, 0.0, 0.05], torch.float32))
        else:
            st["settings"] = {k: c[k] for k in ("temperature", "top_k", "top_p", "min_p")}
        return st

    news = _news(c)
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    parents, tokens, sampled = _trees(c, seed)
    st = dict(case=c, rows=starts[-1], max_new=max(news), starts=ints(starts), parents=ints(parents))
    if c["op"] == "tree":
        st["first"] = (4096 * uniform(c["seqs"])).int()
        return st

    D, lengths, page = c["dim"], _lengths(c), c["page"]
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + 1
    order = torch.randperm(pages, device=dev, generator=gen).to(torch.int32)
    table = torch.full((c["seqs"], max(counts)), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    # keys with channels of different size, as projections leave them; values of one size
    cache = torch.empty(pages, c["kv_heads"], page // 32, 36 * D, dtype=torch.uint8, device=dev)
    step = max(1, (1 << 26) // (c["kv_heads"] * page * D))
    channels = (0.5 * normal(c["kv_heads"], 1, 1, D)).exp()
    for p in range(0, pages, step):
        shape = (min(step, pages - p), c["kv_heads"], page // 32, 32, D)
        cache[p:p + step] = _pack(*_quantise(normal(*shape) * channels, normal(*shape)))
    st.update(cache=cache, table=table, lengths=ints(lengths))
    if c["op"] == "attend":
        st["q"] = (1.5 * normal(st["rows"], c["heads"], D)).to(DTYPES[c["dtype"]])
        st["tree"] = ints(_bits(parents, news, -(-max(news) // 32))[0])
    else:
        st["tokens"], st["sampled"] = ints(tokens), ints(sampled)
        st["path"] = min(c["depth"] + 1, max(news))  # tokens of a path, at most
        st["back"] = torch.arange(c["seqs"] + 1, dtype=torch.int32, device=dev) * st["path"]
    return st


# ---- the cache in plain operations ------------------------------------------------------------------------------------

_NIBBLE = [0, 4, 1, 5, 2, 6, 3, 7]  # where element e of a dword lies


def _quantise(k, v):
    """Float32 [..., D] of keys and values -> (key codes, value codes, key scales, value scales [..., D / 32])."""
    out = []
    for x in (k, v):
        groups = x.unflatten(-1, (-1, 32))
        largest = groups.gather(-1, groups.abs().argmax(-1, keepdim=True))
        d = (largest * -0.125).to(torch.bfloat16).to(torch.float16)
        codes = (groups / d.float() + 8.5).floor().clamp(0, 15)
        out.append((torch.where(d == 0, torch.full_like(codes, 8), codes).to(torch.uint8).flatten(-2), d[..., 0]))
    (kc, kd), (vc, vd) = out
    return kc, vc, kd, vd


def _pack(kc, vc, kd, vd):
    """Codes [..., 32, D] and scales [..., 32, D / 32] -> tiles [..., 36 D]."""
    D, lead = kc.shape[-1], kc.shape[:-2]
    k = kc.reshape(-1, 4, 2, 4, D // 32, 4, 8)         # token (rh, u, rl), value (g, j, e)
    k = k.permute(0, 2, 4, 5, 1, 3, 6)              # u g | j rh rl | e
    v = vc.reshape(-1, 4, 8, D // 16, 16).permute(0, 3, 1, 4, 2)  # w | j r | e
    out = []
    for x in (k, v):
        x = x.reshape(-1, D // 64, 4, 64, 8).transpose(2, 3)    # w >> 2, lane, w & 3, e
        nibbles = torch.empty_like(x)
        nibbles[..., _NIBBLE] = x
        out.append((nibbles[..., 0::2] | (nibbles[..., 1::2] << 4)).reshape(x.shape[0], 16 * D))
    out.append(kd.reshape(-1, D).view(torch.uint8))
    out.append(vd.transpose(-1, -2).reshape(-1, D).view(torch.uint8))
    return torch.cat(out, -1).view(*lead, 36 * D)


def _unpack(tiles):
    """What _pack packed."""
    D, lead = tiles.shape[-1] // 36, tiles.shape[:-1]
    out = []
    for part in (tiles[..., :16 * D], tiles[..., 16 * D:32 * D]):
        x = part.reshape(-1, D // 64, 64, 4, 4)
        x = torch.stack([x & 15, x >> 4], -1).flatten(-2)[..., _NIBBLE].transpose(2, 3)  # w >> 2, w & 3, lane, e
        out.append(x)
    k = out[0].reshape(-1, 2, D // 32, 4, 4, 4, 8).permute(0, 4, 1, 5, 2, 3, 6).reshape(*lead, 32, D)
    v = out[1].reshape(-1, D // 16, 4, 16, 8).permute(0, 2, 4, 1, 3).reshape(*lead, 32, D)
    kd = tiles[..., 32 * D:34 * D].contiguous().view(torch.float16).view(*lead, 32, D // 32)
    vd = tiles[..., 34 * D:].contiguous().view(torch.float16).view(*lead, D // 32, 32).transpose(-1, -2)
    return k, v, kd, vd


def _values(codes, scales):
    return ((codes.float() - 8.0).unflatten(-1, (-1, 32)) * scales.float()[..., None]).flatten(-2)


# ---- one pass ---------------------------------------------------------------------------------------------------------


def run(st):
    return {"tree": _run_tree, "attend": _run_attend, "sample": _run_sample, "accept": _run_accept}[st["case"]["op"]](st)


def _run_tree(st):
    if own:
        from gomlx_amd import nn
        return nn.draft_tree(st["parents"], st["first"], starts=st["starts"], max_new=st["max_new"])
    starts, n = st["starts"].long(), st["max_new"]
    dev = starts.device
    step = torch.arange(n, device=dev)
    real = step < (starts[1:] - starts[:-1])[:, None]
    up = torch.where(real, st["parents"].long()[(starts[:-1, None] + step).clamp(max=st["rows"] - 1)], torch.full_like(step, -1))
    # who is reached by one step or none, then by twice as many each time
    reach = ((up[..., None] == step) | (step[:, None] == step)).float()
    for _ in range(max(1, (n - 1).bit_length())):
        reach = (torch.matmul(reach, reach) > 0).float()
    seq = torch.searchsorted(starts, torch.arange(st["rows"], device=dev), right=True) - 1
    rows = reach[seq, torch.arange(st["rows"], device=dev) - starts[seq]].long()
    words = -(-n // 32)
    bits = torch.nn.functional.pad(rows, (0, 32 * words - n)).unflatten(1, (words, 32))
    bits = (bits << torch.arange(32, device=dev)).sum(-1)
    bits = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).int()
    return bits, st["first"][seq] + (rows.sum(-1) - 1).int()


def _run_attend(st):
    c = st["case"]
    if own:
        from gomlx_amd import nn
        return nn.tree_attention(st["q"], st["cache"], st["table"], st["lengths"], st["tree"], starts=st["starts"], max_new=st["max_new"], window=c["window"])
    kv, group, D = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    starts, lengths = st["starts"].long(), st["lengths"].long()
    dev = lengths.device
    tiles = st["cache"][st["table"].clamp(min=0).long()].transpose(1, 2).flatten(2, 3)
    kc, vc, kd, vd = _unpack(tiles)
    keys = _values(kc, kd).flatten(2, 3)      # [sequences, key heads, tokens, D]
    values = _values(vc, vd).flatten(2, 3)
    step = torch.arange(st["max_new"], device=dev)
    rows = starts[:-1, None] + step
    real = rows < starts[1:, None]
    rows = rows.clamp(max=st["rows"] - 1)
    q = st["q"].float()[rows]   # [sequences, new, heads, D]
    q = q.unflatten(2, (kv, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    # bit j of a row: it sees drafted token j; of what it sees, context and tree, the window has the last ones
    bits = ((st["tree"][rows][..., None] >> torch.arange(32, device=dev, dtype=torch.int32)) & 1).flatten(2)[..., :st["max_new"]]
    own_bits = bits.sum(-1)
    if c["window"]:
        later = bits.flip(-1).cumsum(-1).flip(-1)  # with itself
        bits = bits * (later <= c["window"])
    first = lengths - (starts[1:] - starts[:-1])
    token = torch.arange(keys.shape[2], device=dev)
    context = (token < first[:, None])[:, None].expand(-1, len(step), -1)
    if c["window"]:
        context = context & (token >= (first[:, None] + own_bits - c["window"])[..., None])
    at = token - first[:, None]
    drafted = bits.gather(2, at.clamp(0, st["max_new"] - 1)[:, None].expand(-1, len(step), -1)) > 0
    drafted = drafted & ((at >= 0) & (token < lengths[:, None]))[:, None]
    seen = (context | drafted) & real[..., None]
    seen = seen[:, None, :, None, :].expand(-1, -1, -1, group, -1).flatten(2, 3)
    scores = torch.matmul(q, keys.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(D))
    scores = torch.where(seen, scores, torch.full_like(scores, -math.inf))
    largest = scores.amax(-1, keepdim=True)
    p = torch.where(seen, (scores - torch.where(largest == -math.inf, torch.zeros_like(largest), largest)).exp(), torch.zeros_like(scores))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.matmul(p, values).unflatten(2, (-1, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    row = torch.arange(st["rows"], device=dev)
    seq = torch.searchsorted(starts, row, right=True) - 1
    return out[seq, row - starts[seq]].to(st["q"].dtype)


def _run_sample(st):
    s = st["settings"]
    if own:
        from gomlx_amd import nn
        return nn.sample(st["logits"], st["uniform"], probabilities=True, **s)
    x, u = st["logits"].double(), st["uniform"].double()[:, None]
    rows, vocab = x.shape
    t, k, top_p, min_p = (v.double()[:, None] if isinstance(v, torch.Tensor) else torch.full((rows, 1), float(v), dtype=torch.float64, device=x.device)
                          for v in (s["temperature"], s["top_k"], s["top_p"], s["min_p"]))
    greedy = t <= 0
    x, order = x.sort(dim=-1, descending=True, stable=True)  # ties: the lower index first
    y = (x - x[:, :1]) / torch.where(greedy, torch.ones_like(t), t)
    p = y.exp()
    place = torch.arange(vocab, device=x.device)
    p = torch.where((place < torch.where(k <= 0, torch.full_like(k, vocab), k)) & (~greedy | (place == 0)), p, torch.zeros_like(p))
    upto = p.cumsum(-1)
    keep = (upto - p < top_p * upto[:, -1:]) | (top_p >= 1) | (place == 0)
    keep &= (y >= min_p.log()) | (min_p <= 0)
    p = torch.where(keep, p, torch.zeros_like(p))
    p = torch.empty_like(p).scatter_(1, order, p)  # by index again
    del x, y, order, keep
    upto = p.cumsum(-1)
    total = upto[:, -1:]
    token = (upto <= u * total).sum(-1, keepdim=True).clamp(max=vocab - 1)
    return token[:, 0].int(), (p.gather(1, token) / total)[:, 0].float()


def _run_accept(st):
    c = st["case"]
    seqs, page = c["seqs"], c["page"]
    if own:
        from gomlx_amd import nn
        path, token, lengths = nn.kv_cache_accept(st["cache"], st["table"], st["lengths"], st["parents"], st["tokens"], st["sampled"], starts=st["starts"], max_new=st["max_new"])
        k, v = nn.kv_cache_read(st["cache"], st["table"], lengths, starts=st["back"], max_new=st["path"], rows=seqs * st["path"])
        return path, token, lengths, k, v
    starts, lengths = st["starts"].long(), st["lengths"].long()
    dev, n = lengths.device, st["max_new"]
    step = torch.arange(n, device=dev)
    real = step < (starts[1:] - starts[:-1])[:, None]
    rows = (starts[:-1, None] + step).clamp(max=st["rows"] - 1)
    up, word, draw_ = (x.long()[rows] for x in (st["parents"], st["tokens"], st["sampled"]))
    at = torch.zeros(seqs, 1, dtype=torch.long, device=dev)
    going = torch.ones_like(at, dtype=torch.bool)
    path = [at]
    token = draw_.gather(1, at)
    for _ in range(n - 1):
        child = (up == at) & (word == token) & real & (step > at) & going
        going = child.any(-1, keepdim=True)
        at = torch.where(going, child.float().argmax(-1, keepdim=True), at)
        token = draw_.gather(1, at)
        path.append(torch.where(going, at, torch.full_like(at, -1)))
    path = torch.cat(path, 1)
    count = (path >= 0).sum(-1)
    first = lengths - (starts[1:] - starts[:-1])
    # the tiles that a sequence's drafted tokens lie in; past its last one that one again
    tile = first[:, None] // 32 + torch.arange((n + 30) // 32 + 1, device=dev)
    tile = torch.minimum(tile, (lengths[:, None] - 1) // 32)
    where = (st["table"].gather(1, tile * 32 // page).long(), slice(None), tile * 32 % page // 32)
    old = _unpack(st["cache"][where])  # [sequences, tiles, key heads, 32, ...]
    pos = tile[..., None] * 32 + torch.arange(32, device=dev)
    new = pos - first[:, None, None]  # of the drafted tokens
    source = torch.where((new >= 0) & (new < count[:, None, None]), first[:, None, None] + path[torch.arange(seqs, device=dev)[:, None, None], new.clamp(0, n - 1)], pos)
    source = source - first[:, None, None] // 32 * 32  # from the first of the tiles on
    packed = []
    for o in old:
        flat = o.transpose(1, 2).flatten(2, 3)
        moved = flat.gather(2, source.flatten(1)[:, None, :, None].expand(-1, flat.shape[1], -1, flat.shape[3]))
        packed.append(moved.unflatten(2, (-1, 32)).transpose(1, 2))
    st["cache"][where] = _pack(*packed)
    m = st["path"]
    last = (first + count)[:, None] - m + torch.arange(m, device=dev)
    seq = torch.arange(seqs, device=dev).repeat_interleave(m)
    p = last.flatten()
    q = p.clamp(min=0)
    kc, vc, kd, vd = _unpack(st["cache"][st["table"][seq, q // page].long(), :, q % page // 32])
    in_tile = (q % 32)[:, None, None, None]
    back = [_values(*(x.gather(2, in_tile.expand(-1, x.shape[1], 1, x.shape[3]))[:, :, 0] for x in pair)).half() for pair in ((kc, kd), (vc, vd))]
    back = [torch.where((p >= 0)[:, None, None], x, torch.zeros_like(x)) for x in back]
    return path.int(), token[:, 0].int(), (first + count).int(), *back


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------


def _cell(cache, pages, slots, head, D, values):
    """Keys (or values) [tokens, D] in float64 of one key head, each nibble and scale fetched from its address."""
    dev = cache.device
    tiles = cache.shape[2]
    base = ((pages * cache.shape[1] + head) * tiles + slots // 32) * (36 * D)
    t, x = (slots % 32)[:, None], torch.arange(D, device=dev)[None, :]
    if values:
        w, lane, e = x // 16, 16 * (t // 8) + x % 16, t % 8
        code, scale = 16 * D, 34 * D + (x // 32 * 32 + t) * 2
    else:
        u = t // 4 % 2
        w, lane, e = u * (D // 32) + x // 32, 16 * (x % 32 // 8) + 4 * (t // 8) + t % 4, x % 8
        code, scale = 0, 32 * D + (t * (D // 32) + x // 32) * 2
    nibble = e // 2 + 4 * (e % 2)
    at = base[:, None] + code + ((w // 4 * 64 + lane) * 4 + w % 4) * 4 + nibble // 2
    flat = cache.view(-1)
    c = (flat[at].long() >> (4 * (nibble % 2))) & 15
    d = flat.view(torch.float16)[(base[:, None] + scale) // 2].double()
    return (c - 8).double() * d


def _exact_sample(st):
    """Row by row, from the logits' values in order: a token stays if the tokens in front of it weigh too little."""
    tokens, shares = [], []
    settings = {k: v.tolist() if isinstance(v, torch.Tensor) else [v] * st["case"]["rows"] for k, v in st["settings"].items()}
    draws = st["uniform"].tolist()
    for r, row in enumerate(st["logits"]):
        x = row.double()
        t, k, top_p, min_p = (settings[n][r] for n in ("temperature", "top_k", "top_p", "min_p"))
        most = x.max()
        if t <= 0:
            tokens.append(int((x == most).nonzero()[0]))
            shares.append(1.0)
            continue
        y = (x - most) / t
        order = torch.argsort(-x, stable=True)
        if k > 0:
            order = order[:k]
        if top_p < 1:
            share = torch.softmax(y[order], 0)
            in_front = torch.cumsum(share, 0) - share
            order = order[:max(1, int((in_front < top_p).sum()))]
        if min_p > 0:
            order = order[y[order] >= math.log(min_p)]
        order = order.sort().values
        weight = torch.exp(y[order])
        sums = torch.cumsum(weight, 0)
        at = min(int(torch.searchsorted(sums, sums[-1] * draws[r], right=True)), len(order) - 1)
        tokens.append(int(order[at]))
        shares.append(float(weight[at] / sums[-1]))
    dev = st["logits"].device
    return torch.tensor(tokens, dtype=torch.int32, device=dev), torch.tensor(shares, dtype=torch.float64, device=dev)


def exact(case, seed):
    st = prepare(case, seed)
    c = case
    if c["op"] == "sample":
        return _exact_sample(st)
    news = _news(c)
    dev = st["starts"].device
    if c["op"] == "tree":
        bits, depths = _bits(st["parents"].tolist(), news, -(-max(news) // 32))
        first = [p for p, n in zip(st["first"].tolist(), news) for _ in range(n)]
        return torch.tensor(bits, dtype=torch.int32, device=dev), torch.tensor([p + d for p, d in zip(first, depths)], dtype=torch.int32, device=dev)
    D, table, page, kv = c["dim"], st["table"].long(), c["page"], c["kv_heads"]
    lengths, at = _lengths(c), 0
    if c["op"] == "accept":
        up, word, drawn = (st[n].tolist() for n in ("parents", "tokens", "sampled"))
        paths, token, after, ks, vs = [], [], [], [], []
        for b, (n, length) in enumerate(zip(news, lengths)):
            path = [0]
            while True:
                child = [i for i in range(path[-1] + 1, n) if up[at + i] == path[-1] and word[at + i] == drawn[at + path[-1]]]
                if not child:
                    break
                path.append(child[0])
            token.append(drawn[at + path[-1]])
            paths.append(path + [-1] * (max(news) - len(path)))
            after.append(length - n + len(path))
            places = torch.tensor([p for p in range(length - n)] + [length - n + i for i in path], device=dev)[-st["path"]:]
            for out, values in ((ks, False), (vs, True)):
                x = torch.stack([_cell(st["cache"], table[b, places // page], places % page, h, D, values) for h in range(kv)], 1)
                out.append(torch.nn.functional.pad(x, (0, 0, 0, 0, st["path"] - len(places), 0)))
            at += n
        return (*(torch.tensor(v, dtype=torch.int32, device=dev) for v in (paths, token, after)), torch.cat(ks), torch.cat(vs))
    group, outs = c["heads"] // kv, []
    bits = st["tree"].tolist()
    for b, (n, length) in enumerate(zip(news, lengths)):
        q = st["q"][at:at + n].double().view(n, kv, group, D)
        seen = torch.zeros(n, length, dtype=torch.bool)
        for i in range(n):
            places = [length - n + j for j in range(n) if bits[at + i][j // 32] >> (j % 32) & 1]
            left = length if not c["window"] else c["window"]
            places = places[max(0, len(places) - left):]
            seen[i, places] = True
            seen[i, max(0, length - n - (left - len(places))):length - n] = True
        seen = seen.to(dev)
        at += n
        j = torch.arange(length, device=dev)
        pages, slots = table[b, j // page], j % page
        heads = []
        for h in range(kv):
            s = (q[:, h].reshape(n * group, D) @ _cell(st["cache"], pages, slots, h, D, False).t()).view(n, group, length) / math.sqrt(D)
            p = s.masked_fill(~seen[:, None], -math.inf).softmax(-1)
            heads.append((p.view(n * group, length) @ _cell(st["cache"], pages, slots, h, D, True)).view(n, group, D))
        outs.append(torch.stack(heads, 1).view(n, c["heads"], D))
    return torch.cat(outs)
