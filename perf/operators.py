"""Attention over a cache held in 4 bits and what stands around it in a decoder layer, as cases to be timed.

Four operators, in the order in which a serving step calls them:

* rope    ``qk_norm_rope``: an RMS norm of each query and key head with the position rotation in the same pass;
* append  ``kv_cache_append``: keys and values of new tokens into the cache, which holds them in 4 bits
          (``kv_cache_read`` gives back what the cache then stands for);
* attend  ``cached_attention``: softmax attention of the new tokens over the cache, where asked for with the weight that each
          cached token received added to its account;
* evict   ``kv_cache_evict``: of every sequence and key head only the last tokens and those of largest account stay.

With ``own`` false, ``run`` computes them from elementary torch operations in 32 bits; with ``own`` true it calls gomlx_amd.nn.

The cache, uint8 [pages, key heads, tiles of a page, 36 D]: a tile holds 32 tokens of one key head.  A group is 32 neighbouring
values of a head vector; it stands for d (c - 8) with a scale d (float16 of 8 significant bits) and codes c of 4 bits.

    bytes 0 to 16 D       key codes, dwords [w >> 2][lane][w & 3]: w = u D/32 + g, lane = 16 j + r;
                          token 8 (r >> 2) + 4 u + (r & 3), values 32 g + 8 j + e, e = 0 to 7
    bytes 16 D to 32 D    value codes, dwords [w >> 2][lane][w & 3]: lane = 16 j + r; tokens 8 j + e, value 16 w + r
                          (element e of a dword lies in its nibble (e >> 1) + 4 (e & 1))
    bytes 32 D to 34 D    key scales [token][group]
    bytes 34 D to 36 D    value scales [group][token]

Token p of sequence b lies in page ``page_table[b, p // tokens of a page]``.  ``lengths`` counts the tokens of a sequence with
the new ones; rows ``starts[b]`` to ``starts[b + 1]`` of a call's arguments are sequence b's new tokens, the last ones of it.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_LARGEST = 65408.0  # a token with a value of at least this magnitude (or a NaN) in a head's key or value reads as NaN


def listed():
    layer = dict(heads=32, kv_heads=8, dim=128)  # 4096 values as queries, 1024 as keys and as values
    return [
        # One token of one sequence in float32: the smallest call, where latency counts.
        dict(name="rope_rows1", op="rope", dtype="f32", out="f32", rows=1, rot=128, interleaved=False, norm=True, **layer),
        # A prompt behind float32 projections, on to bfloat16 attention.
        dict(name="rope_rows2048", op="rope", dtype="f32", out="bf16", rows=2048, rot=128, interleaved=False, norm=True, **layer),
        # A decode step of 32 sequences of mixed lengths.
        dict(name="append_seqs32", op="append", dtype="bf16", seqs=32, new=1, length=4000, page=64, **layer),
        # Prompts of mixed lengths in one call, beginning anywhere in a page.
        dict(name="append_prompts7", op="append", dtype="f32", seqs=7, new=509, length=1500, page=128, **layer),
        # One sequence, one token, float32: few workgroups' worth of cache.
        dict(name="attend_rows1", op="attend", dtype="f32", seqs=1, new=1, length=2047, page=64, window=0, weights=False, **layer),
        # A decode batch in bfloat16 over caches of mixed lengths.
        dict(name="attend_seqs32", op="attend", dtype="bf16", seqs=32, new=1, length=8192, page=64, window=0, weights=False, **layer),
        # One token over one very long cache: the work is split along it and joined.
        dict(name="attend_long", op="attend", dtype="bf16", seqs=1, new=1, length=131072, page=256, window=0, weights=False, **layer),
        # A decode batch whose cache will be evicted from: accounts of the weights are kept.
        dict(name="attend_account", op="attend", dtype="bf16", seqs=16, new=1, length=4096, page=64, window=0, weights=True, **layer),
        # A prompt's second half: matrix products bound it.
        dict(name="attend_prompt", op="attend", dtype="bf16", seqs=1, new=2048, length=4096, page=64, window=0, weights=False, **layer),
        # Ragged prompts in float32 with a window and accounts, smaller heads, one key head a query head.
        dict(name="attend_ragged", op="attend", dtype="f32", seqs=5, new=301, length=1111, page=32, window=500, weights=True, heads=12, kv_heads=12, dim=64),
        # One sequence over its budget.
        dict(name="evict_seq1", op="evict", dtype="bf16", seqs=1, new=1, length=4096, page=64, keep=2048, recent=256, **layer),
        # A batch of long sequences, a quarter of the longest kept.
        dict(name="evict_seqs16", op="evict", dtype="bf16", seqs=16, new=1, length=16384, page=128, keep=4096, recent=512, **layer),
    ]


_MAX_FLOPS = 1.0e11   # of the largest listed cases (the prompt
_MAX_BYTES = 5.0e8    # the batch that is evicted from)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges."""
    while True:
        op = rng.choice(("rope", "append", "attend", "attend", "attend", "attend", "evict"))
        dim = rng.choice((64, 128, 128, 256))
        kv = rng.choice((1, 2, 4, 8, 8, 12, 16))
        c = dict(op=op, dtype=rng.choice(("f32", "bf16", "bf16")), heads=kv * rng.choice((1, 2, 3, 4, 4, 7, 8)), kv_heads=kv, dim=dim)
        if op == "rope":
            c.update(out=rng.choice(("f32", "bf16")), rows=_log(rng, 1, 4096), rot=rng.choice((dim, dim, dim // 2)), interleaved=rng.random() < 0.4, norm=rng.random() < 0.7)
        else:
            prompt = rng.random() < 0.5 and op != "evict"
            c.update(seqs=_log(rng, 1, 8 if prompt else 48), new=_log(rng, 2, 2048) if prompt else 1, page=rng.choice((32, 64, 96, 128, 256)))
            c["length"] = c["new"] + _log(rng, 1, 30000)
        if op == "attend":
            c.update(window=_log(rng, 16, c["length"]) if rng.random() < 0.25 else 0, weights=rng.random() < 0.3)
        if op == "evict":
            c["keep"] = max(1, int(c["length"] * rng.uniform(0.1, 0.8)))
            c["recent"] = int(c["keep"] * rng.uniform(0.0, 0.9))
        w = work(c)
        # (the plain form holds keys and values in float32 and, of a prompt, every score)
        cells = c.get("seqs", 0) * c.get("length", 0) * kv * dim
        scores = c.get("seqs", 0) * c.get("length", 0) * c["heads"] * c.get("new", 0)
        if w["flops"] <= _MAX_FLOPS and w["bytes"] <= _MAX_BYTES and cells <= 3.0e8 and scores <= 4.0e8:
            return c


def _news(c):
    """New tokens of each sequence: the longest first, odd steps down to half of it."""
    return [max(1, c["new"] - b * c["new"] // (2 * c["seqs"])) for b in range(c["seqs"])]


def _lengths(c):
    """Tokens of each sequence with the new ones: the longest first, down to a quarter of it."""
    return [max(n, c["length"] - 3 * b * c["length"] // (4 * c["seqs"])) for b, n in enumerate(_news(c))]


def work(case):
    c, D = case, case["dim"]
    size = {"f32": 4, "bf16": 2}
    if c["op"] == "rope":
        values = c["rows"] * (c["heads"] + c["kv_heads"]) * D
        return {"bytes": float(values * (size[c["dtype"]] + size[c["out"]]) + c["rows"] * c["rot"] * 4), "flops": 6.0 * values}
    rows, token = sum(_news(c)), 36 * D // 32 * c["kv_heads"]  # bytes of a cached token
    if c["op"] == "append":  # and the new tokens read back
        values = 2 * rows * c["kv_heads"] * D
        return {"bytes": float(values * (size[c["dtype"]] + 2) + 2 * rows * token), "flops": 4.0 * values}
    if c["op"] == "evict":
        lengths = _lengths(c)
        kept = sum(min(n, c["keep"]) for n in lengths)
        return {"bytes": float(4 * c["kv_heads"] * (sum(lengths) + 2 * kept) + 3 * kept * token + 4 * kept * c["kv_heads"] * D), "flops": float(c["kv_heads"] * sum(lengths))}
    pairs = tokens = 0
    for n, length in zip(_news(c), _lengths(c)):
        span = min(length, c["window"]) if c["window"] else length
        seen = [min(p + 1, span) for p in range(length - n, length)]
        pairs += sum(seen)
        tokens += min(length, max(seen) + n - 1)
    return {"bytes": float(tokens * token + 2 * rows * c["heads"] * D * size[c["dtype"]] + (8 * tokens * c["kv_heads"] if c["weights"] else 0)),
            "flops": 4.0 * D * c["heads"] * pairs}


# ---- the inputs ------------------------------------------------------------------------------------------------------


def prepare(case, seed):
    c = dict(case)
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    D, dtype = c["dim"], DTYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(shape, device=dev, generator=gen)

    if c["op"] == "rope":
        # queries and keys as one projection leaves them, positions up to 32768 (all of a prompt's in order), 64-bit angles
        wide = normal(c["rows"], (c["heads"] + 2 * c["kv_heads"]) * D).to(dtype)
        q = wide[:, :c["heads"] * D].view(c["rows"], c["heads"], D)
        k = wide[:, c["heads"] * D:(c["heads"] + c["kv_heads"]) * D].view(c["rows"], c["kv_heads"], D)
        first = torch.randint(0, 32768 - c["rows"], (1,), device=dev, generator=gen, dtype=torch.int32)
        rates = 500000.0 ** (-torch.arange(0, c["rot"], 2, device=dev, dtype=torch.float64) / c["rot"])
        angles = torch.arange(32768, device=dev, dtype=torch.float64)[:, None] * rates
        st = dict(case=c, q=q, k=k, positions=first + torch.arange(c["rows"], device=dev, dtype=torch.int32), cos=angles.cos().float(), sin=angles.sin().float())
        st["gains"] = [1.0 + 0.1 * normal(D) for _ in range(2)] if c["norm"] else None
        return st

    news, lengths, page = _news(c), _lengths(c), c["page"]
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
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    rows = starts[-1]
    st = dict(case=c, cache=cache, table=table, lengths=torch.tensor(lengths, dtype=torch.int32, device=dev), rows=rows, max_new=max(news),
              starts=torch.tensor(starts, dtype=torch.int32, device=dev) if c["new"] > 1 else None)
    if c["op"] == "append":
        k, v = normal(2, rows, c["kv_heads"], D).to(dtype)
        st.update(k=k, v=v)
    elif c["op"] == "attend":
        st["q"] = (1.5 * normal(rows, c["heads"], D)).to(dtype)
        st["weights"] = 0.01 * normal(pages, c["kv_heads"], page).square() if c["weights"] else None
    else:
        # accounts as steps of attention leave them: a few large ones, many small, some exactly equal
        w = (2.0 * normal(pages, c["kv_heads"], page)).exp()
        st["weights"] = torch.where(w < 0.05, torch.zeros_like(w), w)
    return st


# ---- the cache in plain operations ------------------------------------------------------------------------------------

_NIBBLE = [0, 4, 1, 5, 2, 6, 3, 7]  # where element e of a dword lies


def _quantise(k, v):
    """Float32 [..., D] of keys and values -> (key codes, value codes, key scales, value scales [..., D / 32])."""
    good = ((k.abs() < _LARGEST) & (v.abs() < _LARGEST)).all(-1, keepdim=True)
    out = []
    for x in (k, v):
        groups = torch.where(good, x, torch.zeros_like(x)).unflatten(-1, (-1, 32))
        largest = groups.gather(-1, groups.abs().argmax(-1, keepdim=True))
        d = (largest * -0.125).to(torch.bfloat16).to(torch.float16)
        codes = (groups / d.float() + 8.5).floor().clamp(0, 15)
        out.append((torch.where(d == 0, torch.full_like(codes, 8), codes).to(torch.uint8).flatten(-2), d[..., 0]))
    (kc, kd), (vc, vd) = out
    return kc, vc, torch.where(good, kd, torch.full_like(kd, math.nan)), vd


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


def _dense(cache, table):
    """The tiles of every sequence in order: [sequences, key heads, tiles, 36 D]."""
    return cache[table.clamp(min=0).long()].transpose(1, 2).flatten(2, 3)


def _row_of(st):
    """(sequence, position) of every row of the call."""
    lengths = st["lengths"].long()
    if st["starts"] is None:
        return torch.arange(st["rows"], device=lengths.device), lengths - 1
    starts = st["starts"].long()
    rows = torch.arange(st["rows"], device=lengths.device)
    seq = torch.searchsorted(starts, rows, right=True) - 1
    return seq, lengths[seq] - starts[seq + 1] + rows


def _starts(st):
    return torch.arange(st["rows"] + 1, device=st["lengths"].device) if st["starts"] is None else st["starts"].long()


def _read(st, seq, pos):
    """Keys and values [rows, key heads, D] at positions of sequences, in the float16 numbers that they are."""
    page = st["case"]["page"]
    tiles = st["cache"][st["table"][seq, pos // page].long(), :, pos % page // 32]
    kc, vc, kd, vd = _unpack(tiles)
    at = (pos % 32)[:, None, None, None]
    return [_values(*(x.gather(2, at.expand(-1, x.shape[1], 1, x.shape[3]))[:, :, 0] for x in pair)).half() for pair in ((kc, kd), (vc, vd))]


# ---- one pass ---------------------------------------------------------------------------------------------------------


def run(st):
    return {"rope": _run_rope, "append": _run_append, "attend": _run_attend, "evict": _run_evict}[st["case"]["op"]](st)


def _run_rope(st):
    c = st["case"]
    if own:
        from gomlx_amd import nn
        norms = [nn.RMSNorm(gain=g, epsilon=1e-6) for g in st["gains"]] if c["norm"] else [None, None]
        return nn.qk_norm_rope(st["q"], st["k"], st["positions"], st["cos"], st["sin"], q_norm=norms[0], k_norm=norms[1], interleaved=c["interleaved"], dtype=DTYPES[c["out"]])
    out = []
    at = st["positions"].long()
    cos, sin = st["cos"][at][:, None], st["sin"][at][:, None]
    for i, x in enumerate((st["q"], st["k"])):
        y = x.float()
        if c["norm"]:
            y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + 1e-6) * st["gains"][i]
        turned, rest = y[..., :c["rot"]], y[..., c["rot"]:]
        a, b = (turned[..., 0::2], turned[..., 1::2]) if c["interleaved"] else turned.chunk(2, -1)
        pair = (a * cos - b * sin, a * sin + b * cos)
        turned = torch.stack(pair, -1).flatten(-2) if c["interleaved"] else torch.cat(pair, -1)
        out.append(torch.cat([turned, rest], -1).to(DTYPES[c["out"]]))
    return tuple(out)


def _run_append(st):
    c = st["case"]
    if own:
        from gomlx_amd import nn
        nn.kv_cache_append(st["cache"], st["k"], st["v"], st["table"], st["lengths"], starts=st["starts"], max_new=st["max_new"])
        return nn.kv_cache_read(st["cache"], st["table"], st["lengths"], starts=st["starts"], max_new=st["max_new"], rows=st["rows"])
    starts, lengths, page = _starts(st), st["lengths"].long(), c["page"]
    first = lengths - (starts[1:] - starts[:-1])
    new = _quantise(st["k"].float(), st["v"].float())
    # the tiles that a sequence's new tokens lie in; past its last one that one again
    tile = first[:, None] // 32 + torch.arange((st["max_new"] + 30) // 32 + 1, device=lengths.device)
    tile = torch.minimum(tile, (lengths[:, None] - 1) // 32)
    where = (st["table"].gather(1, tile * 32 // page).long(), slice(None), tile * 32 % page // 32)
    old = st["cache"][where]  # [sequences, tiles, key heads, 36 D]
    pos = tile[..., None] * 32 + torch.arange(32, device=lengths.device)
    fresh = (pos >= first[:, None, None])[:, :, None, :, None] & (pos < lengths[:, None, None])[:, :, None, :, None]
    row = (pos - first[:, None, None] + starts[:-1, None, None]).clamp(0, st["rows"] - 1)
    st["cache"][where] = _pack(*(torch.where(fresh, n[row].transpose(2, 3), o) for n, o in zip(new, _unpack(old))))
    return tuple(_read(st, *_row_of(st)))


def _run_attend(st):
    c = st["case"]
    if own:
        from gomlx_amd import nn
        out = nn.cached_attention(st["q"], st["cache"], st["table"], st["lengths"], starts=st["starts"], max_new=st["max_new"], window=c["window"], weights=st["weights"])
        return (out, st["weights"]) if c["weights"] else out
    kv, group, D, page = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"], c["page"]
    seq, pos = _row_of(st)
    starts, lengths = _starts(st), st["lengths"].long()
    kc, vc, kd, vd = _unpack(_dense(st["cache"], st["table"]))
    keys = _values(kc, kd).flatten(2, 3)      # [sequences, key heads, tokens, D]
    values = _values(vc, vd).flatten(2, 3)
    step = torch.arange(st["max_new"], device=lengths.device)
    rows = starts[:-1, None] + step
    real = rows < starts[1:, None]
    q = st["q"].float()[rows.clamp(max=st["rows"] - 1)]   # [sequences, new, heads, D]
    q = q.unflatten(2, (kv, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    at = (lengths - (starts[1:] - starts[:-1]))[:, None] + step
    token = torch.arange(keys.shape[2], device=lengths.device)
    seen = (token <= at[..., None]) & real[..., None]
    if c["window"]:
        seen &= token > at[..., None] - c["window"]
    seen = seen[:, None, :, None, :].expand(-1, -1, -1, group, -1).flatten(2, 3)
    scores = torch.matmul(q, keys.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(D))
    scores = torch.where(seen, scores, torch.full_like(scores, -math.inf))
    largest = scores.amax(-1, keepdim=True)
    p = torch.where(seen, (scores - torch.where(largest == -math.inf, torch.zeros_like(largest), largest)).exp(), torch.zeros_like(scores))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.matmul(p, values).unflatten(2, (-1, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    out = out[seq, torch.arange(st["rows"], device=seq.device) - starts[seq]].to(st["q"].dtype)
    if not c["weights"]:
        return out
    account = p.sum(2)  # [sequences, key heads, tokens]; tokens past a sequence's end add nothing, to page 0 where there is none
    pages = st["table"].clamp(min=0).long()
    inside = token < lengths[:, None]
    account = torch.where(inside[:, None], account, torch.zeros_like(account)).unflatten(2, (-1, page)).transpose(1, 2)
    st["weights"].index_add_(0, pages.flatten(), account.flatten(0, 1))
    return out, st["weights"]


def _run_evict(st):
    c = st["case"]
    seqs, keep, recent, page = c["seqs"], c["keep"], c["recent"], c["page"]
    dev = st["lengths"].device
    if own:
        from gomlx_amd import nn
        kept, lengths = nn.kv_cache_evict(st["cache"], st["weights"], st["table"], st["lengths"], keep, recent)
        starts = torch.arange(seqs + 1, device=dev, dtype=torch.int32) * keep
        k, v = nn.kv_cache_read(st["cache"], st["table"], lengths, starts=starts, max_new=keep, rows=seqs * keep)
        return kept, lengths, k, v, st["weights"]
    lengths, pages = st["lengths"].long(), st["table"].clamp(min=0).long()
    most = st["table"].shape[1] * page
    weights = st["weights"][pages].transpose(1, 2).flatten(2)  # [sequences, key heads, tokens]
    token = torch.arange(most, device=dev)
    last = (token >= lengths[:, None] - recent) & (token < lengths[:, None])
    # the recent ones first, then by weight, then what lies past the end
    order = torch.where((token < lengths[:, None])[:, None], weights, torch.full_like(weights, -math.inf))
    order = torch.where(last[:, None], torch.full_like(order, math.inf), order)
    best = order.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    if best.shape[-1] < keep:  # (a budget past the table's end)
        best = torch.nn.functional.pad(best, (0, keep - best.shape[-1]), value=most)
    kept = torch.where(torch.arange(keep, device=dev) < lengths[:, None, None].clamp(max=keep), best, torch.full_like(best, most)).sort(-1).values
    here = kept < most
    source = torch.where(here, kept, torch.arange(keep, device=dev).clamp(max=most - 1))
    # in place: the first tokens of every sequence become the kept ones (tiles and tokens of pages that a short sequence does
    # not have are replaced by its first tile and token)
    tiles = _dense(st["cache"], st["table"])
    count = min(-(-keep // 32), tiles.shape[2])
    n, packed = min(keep, most), []
    for x in _unpack(tiles):
        flat = x.flatten(2, 3)
        moved = flat[:, :, :count * 32].clone()
        moved[:, :, :n] = flat.gather(2, source[:, :, :n, None].expand(-1, -1, -1, flat.shape[3]))
        packed.append(moved.unflatten(2, (count, 32)))
    account = weights.clone()
    account[:, :, :n] = weights.gather(2, source[:, :, :n])
    for buffer, new, unit in ((st["cache"], _pack(*packed), 32), (st["weights"], account, 1)):
        at = torch.arange(new.shape[2], device=dev) * unit
        at = torch.where(st["table"][:, at // page] >= 0, at, torch.zeros_like(at))
        new = new.transpose(1, 2)[torch.arange(seqs, device=dev)[:, None], at // unit]
        buffer[pages.gather(1, at // page), :, at % page // unit] = new
    seq = torch.arange(seqs, device=dev).repeat_interleave(keep)
    pos = (lengths.clamp(max=keep)[:, None] - keep + torch.arange(keep, device=dev)).flatten()
    k, v = (torch.where((pos >= 0)[:, None, None], x, torch.zeros_like(x)) for x in _read(st, seq, pos.clamp(min=0)))
    return torch.where(here, kept, torch.full_like(kept, -1)).int(), lengths.clamp(max=keep).int(), k, v, st["weights"]


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


def exact(case, seed):
    st = prepare(case, seed)
    c, D = case, case["dim"]
    if c["op"] == "rope":
        out = []
        for i, x in enumerate((st["q"], st["k"])):
            x = x.double()
            if c["norm"]:
                x = x * (x.square().sum(-1, keepdim=True) / D + 1e-6).rsqrt() * st["gains"][i].double()
            cos, sin = (t[st["positions"].long()].double()[:, None] for t in (st["cos"], st["sin"]))
            half = torch.arange(c["rot"] // 2, device=x.device)
            a, b = (2 * half, 2 * half + 1) if c["interleaved"] else (half, half + c["rot"] // 2)
            y = x.clone()
            y[..., a] = x[..., a] * cos - x[..., b] * sin
            y[..., b] = x[..., a] * sin + x[..., b] * cos
            out.append(y)
        return tuple(out)
    if c["op"] == "append":
        out = []
        for x in (st["k"].double(), st["v"].double()):
            g = x.view(*x.shape[:-1], D // 32, 32)
            m = g.gather(-1, g.abs().argmax(-1, keepdim=True))
            d = (-m / 8).float().bfloat16().half().double()
            n = torch.floor(g / d + 0.5).clamp(-8, 7)
            out.append(torch.where(d == 0, torch.zeros_like(g), n * d).flatten(-2))
        return tuple(out)
    table, page, kv = st["table"].long(), c["page"], c["kv_heads"]
    if c["op"] == "evict":
        kept, ks, vs, account = [], [], [], st["weights"].double().clone()
        for b, length in enumerate(_lengths(c)):
            pos = torch.arange(length, device=table.device)
            w = st["weights"][table[b, pos // page], :, pos % page].t()  # [key heads, tokens]
            if length > c["keep"]:
                old = length - c["recent"]
                order = torch.sort(w[:, :old], dim=-1, descending=True, stable=True).indices[:, :c["keep"] - c["recent"]]
                keep = torch.cat([order.sort(-1).values, torch.arange(old, length, device=table.device).expand(kv, -1)], -1)
            else:
                keep = pos.expand(kv, -1)
            n = keep.shape[1]
            kept.append(torch.nn.functional.pad(keep, (0, c["keep"] - n), value=-1).int())
            for h in range(kv):
                account[table[b, pos[:n] // page], h, pos[:n] % page] = w[h, keep[h]].double()
            for out, values in ((ks, False), (vs, True)):
                x = torch.stack([_cell(st["cache"], table[b, keep[h] // page], keep[h] % page, h, D, values) for h in range(kv)], 1)
                out.append(torch.nn.functional.pad(x, (0, 0, 0, 0, c["keep"] - n, 0)))
        lengths = torch.tensor([min(n, c["keep"]) for n in _lengths(c)], dtype=torch.int32, device=table.device)
        return torch.stack(kept), lengths, torch.cat(ks), torch.cat(vs), account
    group, at, outs = c["heads"] // kv, 0, []
    account = st["weights"].double().clone() if c["weights"] else None
    for n, length, b in zip(_news(c), _lengths(c), range(c["seqs"])):
        q = st["q"][at:at + n].double().view(n, kv, group, D)
        at += n
        j = torch.arange(length, device=table.device)
        i = torch.arange(length - n, length, device=table.device)
        hidden = j[None] > i[:, None]
        if c["window"]:
            hidden |= j[None] <= i[:, None] - c["window"]
        pages, slots = table[b, j // page], j % page
        heads = []
        for h in range(kv):
            s = (q[:, h].reshape(n * group, D) @ _cell(st["cache"], pages, slots, h, D, False).t()).view(n, group, length) / math.sqrt(D)
            p = s.masked_fill(hidden[:, None], -math.inf).softmax(-1)
            heads.append((p.view(n * group, length) @ _cell(st["cache"], pages, slots, h, D, True)).view(n, group, D))
            if c["weights"]:
                account[pages, h, slots] += p.sum((0, 1))
        outs.append(torch.stack(heads, 1).view(n, c["heads"], D))
    out = torch.cat(outs)
    return (out, account) if c["weights"] else out
