"""Serving several sequences from one cache of 4-bit pages: what the operators compute, and on which sizes they are timed.

Three operators (fwb.kv4, fwb.sampling), in a plain form written with elementary torch operations and as the library's
kernels:

- appending new tokens to a paged cache whose keys and values are held in 4 bits: queries and keys are rotated by position,
  keys and values quantised in blocks of 32 and written to their pages (and read back, to return what the cache then holds);
- attention of each sequence's newest tokens over its pages;
- sampling of a token per row with temperature, top-k, top-p and min-p from given uniform numbers.

A page of the cache is, for each head, a line of tiles of 16 positions; a tile holds the codes of its keys, their scales, the
codes of its values and their scales. A block of 32 values has one fp16 scale d and codes 0..15 that stand for (code - 8) * d.
Lengths and page tables follow from the case alone, so that `work` counts what a pass needs; values follow from the seed.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ESIZE = {"f32": 4, "f16": 2, "bf16": 2}
HEADS = {"8b": (32, 8, 128), "70b": (64, 8, 128), "small": (4, 2, 128), "tp8": (8, 8, 128), "tiny": (6, 6, 48)}
TILE = 16


def _fwb():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "forword.c_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from fwb import kv4, sampling
    return kv4, sampling


def _attn(name, dtype, heads, seqs, queries, length, page, ragged):
    return {"name": name, "op": "attention", "dtype": dtype, "heads": heads, "seqs": seqs, "queries": queries, "length": length,
            "page": page, "ragged": ragged}


def _append(name, dtype, heads, seqs, queries, length, page, ragged, halves):
    return {"name": name, "op": "append", "dtype": dtype, "heads": heads, "seqs": seqs, "queries": queries, "length": length,
            "page": page, "ragged": ragged, "halves": halves}


def _sample(name, dtype, rows, vocab, filters):
    return {"name": name, "op": "sample", "dtype": dtype, "rows": rows, "vocab": vocab, "filters": filters}


def listed():
    return [
        # one layer of the decode step after a short question, fp32 activations as the 8B model's: latency
        _attn("attn_f32_short", "f32", "8b", 1, 1, 200, 16, False),
        # the same late in a long context
        _attn("attn_f16_long", "f16", "8b", 1, 1, 8000, 64, False),
        # five sequences of the small model's six 48-wide heads, odd lengths
        _attn("attn_f32_tiny", "f32", "tiny", 5, 1, 251, 32, True),
        # checking seven drafted tokens of nine sequences
        _attn("attn_bf16_drafts", "bf16", "8b", 9, 7, 4099, 16, True),
        # a server's batch on the 70B shape, ragged contexts
        _attn("attn_bf16_batch", "bf16", "70b", 64, 1, 8191, 64, True),
        # a chunk of 512 prompt tokens at the end of a long prompt
        _attn("attn_f16_chunk", "f16", "8b", 1, 512, 8191, 128, False),
        # the step of a server's batch: one token of each of 64 sequences
        _append("append_f16_step", "f16", "8b", 64, 1, 1500, 16, True, False),
        # a prompt of 2048 tokens into an empty cache, fp32 activations
        _append("append_f32_prompt", "f32", "8b", 1, 2048, 2048, 64, False, False),
        # a padded batch of prompt chunks, halves rotated against each other
        _append("append_bf16_chunks", "bf16", "70b", 7, 333, 2000, 32, True, True),
        # the next token of one sequence: latency
        _sample("sample_f32_one", "f32", 1, 128256, "all"),
        # a server's batch, every row with settings of its own (some greedy, some without filters)
        _sample("sample_bf16_batch", "bf16", 64, 128256, "mixed"),
        # many rows of the small vocabulary, temperature alone
        _sample("sample_f16_open", "f16", 256, 32000, "none"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "sample"])
    cases = listed()
    if op == "attention":
        flops, size = _work(cases[5])["flops"], _work(cases[4])["bytes"]
        while True:
            q = rng.choice([1, 1, 1, _log(rng, 2, 8), _log(rng, 16, 512)])
            c = _attn("", rng.choice(["f32", "f16", "bf16"]), rng.choice(sorted(HEADS)), _log(rng, 1, 64), q,
                      q - 1 + _log(rng, 1, 32768), rng.choice([16, 32, 64, 128]), rng.random() < 0.5)
            w = _work(c)
            nh = HEADS[c["heads"]][0]
            if (w["flops"] * (2 if c["dtype"] == "f32" else 1) <= flops and w["bytes"] <= size
                    and c["seqs"] * nh * c["queries"] * c["length"] <= 1 << 28):
                break
    elif op == "append":
        largest = _work(cases[8])["bytes"]
        while True:
            c = _append("", rng.choice(["f32", "f16", "bf16"]), rng.choice(sorted(HEADS)), _log(rng, 1, 64),
                        rng.choice([1, _log(rng, 2, 2048)]), 0, rng.choice([16, 32, 64, 128]), rng.random() < 0.5, rng.random() < 0.5)
            c["length"] = c["queries"] - 1 + _log(rng, 1, 8192)
            if _work(c)["bytes"] <= largest and c["seqs"] * c["length"] <= 1 << 17:
                break
    else:
        while True:
            c = _sample("", rng.choice(["f32", "f16", "bf16"]), _log(rng, 1, 256), _log(rng, 1000, 128256),
                        rng.choice(["none", "k", "p", "min", "all", "mixed"]))
            if c["rows"] * c["vocab"] <= 64 * 128256:
                break
    del c["name"]
    return c


# --- lengths and page tables: from the case alone ---------------------------------------------------
def _lengths(c):
    """(length of each sequence with its new tokens, new tokens of each): the first has all, others fewer where ragged."""
    n, nq = c["seqs"], c["queries"]
    if not c["ragged"]:
        return [c["length"]] * n, [nq] * n
    room = c["length"] - nq
    new = [nq - (i * 7 % n) * (nq - 1) // n for i in range(n)] if c["op"] == "append" else [nq] * n
    return [new[i] + room - (i * 37 % n) * room // n for i in range(n)], new


def _pages(c):
    """(page table [seqs][most pages], pages of the cache): the sequences' pages lie scattered, two belong to nobody."""
    lens, _ = _lengths(c)
    need = [-(-n // c["page"]) for n in lens]
    rng = random.Random("%d %d %d" % (c["seqs"], c["length"], c["page"]))
    free = list(range(sum(need) + 2))
    rng.shuffle(free)
    table = []
    for n in need:
        table.append([free.pop() for _ in range(n)] + [0] * (max(need) - n))
    return table, sum(need) + 2


def _work(c):
    if c["op"] == "sample":
        return {"bytes": c["rows"] * (c["vocab"] * ESIZE[c["dtype"]] + 28), "flops": 4 * c["rows"] * c["vocab"]}
    nh, nkv, hd = HEADS[c["heads"]]
    e, (lens, new) = ESIZE[c["dtype"]], _lengths(c)
    row = nkv * 2 * (hd // 2 + 2 * -(-hd // 32))   # a position of the cache, in bytes
    if c["op"] == "attention":
        nq = c["queries"]
        pairs = sum(nq * n - nq * (nq - 1) // 2 for n in lens)
        return {"bytes": sum(lens) * row + c["seqs"] * nq * nh * (2 * hd * e + 4), "flops": 4 * pairs * nh * hd}
    # queries read and written, keys and values read, written as codes, and returned as values
    tokens = sum(new)
    return {"bytes": tokens * ((2 * nh + 4 * nkv) * hd * e + 2 * row) + sum(new) * hd * 4,
            "flops": tokens * (nh + nkv) * hd * 3}


def work(case):
    return _work(case)


# --- the cache's format ---------------------------------------------------------------------------
def _blocks(hd):
    return -(-hd // 32)


def _where(hd, device):
    """For each position of a tile and each dimension: the byte of its row that holds its code, and the bits' place, of keys
    [hd] and of values [16, hd]."""
    nb = _blocks(hd)
    d = torch.arange(hd, device=device)
    b, r = d // 32, d % 32
    c, i = r // 8, r % 8
    nib = i // 2 + 4 * (i % 2)
    k = (c * 4 * nb + b * 4 + nib // 2, 4 * (nib % 2))
    p = torch.arange(TILE, device=device)[:, None]
    g, i = r // 4, r % 4
    v = ((g ^ (4 * (p // 2 % 2))) * 2 * nb + 2 * b + i // 2, (4 * (i % 2)).expand(TILE, hd))
    return k, v


def _values(tiles, hd):
    """Keys and values [..., 16, hd] in fp32 that tiles [..., tile bytes] stand for."""
    nb = _blocks(hd)
    lead = tiles.shape[:-1]
    codes, scales = TILE * 16 * nb, TILE * 2 * nb
    (kb, ks), (vb, vs) = _where(hd, tiles.device)
    got = []
    for at, byte, shift in ((0, kb.expand(TILE, hd), ks.expand(TILE, hd)), (codes + scales, vb, vs)):
        rows = tiles[..., at:at + codes].reshape(*lead, TILE, 16 * nb)
        code = (torch.gather(rows, -1, byte.expand(*lead, TILE, hd)).int() >> shift) & 15
        d = tiles[..., at + codes:at + codes + scales].contiguous().view(torch.float16).reshape(*lead, TILE, nb).float()
        got.append((code - 8).float() * torch.repeat_interleave(d, 32, -1)[..., :hd])
    return got


def _quantise(y):
    """Codes [..., hd] and fp16 scales [..., blocks] of fp32 values: the value of the largest magnitude (the positive one of
    two) stands at -8 scales, the others at the nearest code, upwards from the middle."""
    hd = y.shape[-1]
    nb = _blocks(hd)
    y = torch.nn.functional.pad(y, (0, 32 * nb - hd)).reshape(*y.shape[:-1], nb, 32)
    hi, lo = y.amax(-1), y.amin(-1)
    d = (torch.where(hi >= -lo, hi, lo) * -0.125).clamp(-65504, 65504).half()
    by = d.double()[..., None]
    code = torch.where(by != 0, torch.floor(y.double() / by + 8.5).clamp(0, 15), 8.0)
    return code.int().flatten(-2)[..., :hd], d


def _packed(code, at, hd):
    """Rows [..., 16 * blocks] of bytes from codes [..., hd]; at: (byte, shift) of each code, [..., hd]. What a row holds past
    hd stands for zeros."""
    row = torch.zeros(*code.shape[:-1], 16 * _blocks(hd), dtype=torch.int32, device=code.device)
    row.scatter_add_(-1, at[0].expand(code.shape), code << at[1].int().expand(code.shape))
    return row


def _places(c, pages, pos, hd):
    """(first byte of each token's tile for each head [..., heads], place in the tile [...]) of positions pos [seqs, n]."""
    nkv = HEADS[c["heads"]][1]
    tile_bytes = 576 * _blocks(hd)
    page = torch.gather(pages.long(), 1, (pos // c["page"]).clamp(0, pages.shape[1] - 1))
    line = (page[..., None] * nkv + torch.arange(nkv, device=pages.device)) * (c["page"] // TILE)
    return (line + (pos % c["page"] // TILE)[..., None]) * tile_bytes, pos % TILE


def _store(c, cache, pages, pos, ok, k, v):
    """Rows k and v [seqs, n, heads, hd] (fp32) to positions pos of the cache where ok."""
    hd = HEADS[c["heads"]][2]
    nb = _blocks(hd)
    (kb, ks), (vb, vs) = _where(hd, cache.device)
    first, p = _places(c, pages, pos, hd)
    first, p, k, v = first[ok], p[ok], k[ok], v[ok]
    codes, scales = TILE * 16 * nb, TILE * 2 * nb
    flat = cache.view(-1)
    for at, x, place in ((0, k, (kb, ks)), (codes + scales, v, (vb[p][:, None], vs[p][:, None]))):
        code, d = _quantise(x)
        spare = torch.full((*code.shape[:-1], 32 * nb), 8, dtype=torch.int32, device=code.device)
        spare[..., :hd] = code
        (ekb, eks), (evb, evs) = _where(32 * nb, cache.device)
        row = _packed(spare, (ekb, eks) if at == 0 else (evb[p][:, None], evs[p][:, None]), 32 * nb)
        to = first[..., None] + at + p[:, None, None] * 16 * nb + torch.arange(16 * nb, device=cache.device)
        flat[to] = row.to(torch.uint8)
        to = first[..., None] + at + codes + p[:, None, None] * 2 * nb + torch.arange(2 * nb, device=cache.device)
        flat[to] = d.contiguous().view(torch.uint8).reshape(*d.shape[:-1], 2 * nb)


def _load(c, cache, pages, start, n, lens):
    """Keys and values [seqs, n, heads, hd] (fp32) of n positions from start[s] on; 0 at and past a length."""
    nkv, hd = HEADS[c["heads"]][1:]
    pos = start.long()[:, None] + torch.arange(n, device=cache.device)
    ok = ((pos >= 0) & (pos < lens.long()[:, None]))[..., None, None]
    first, p = _places(c, pages, pos.clamp_min(0), hd)
    tiles = cache.view(-1, 576 * _blocks(hd))[first // (576 * _blocks(hd))]
    at = p[..., None, None, None].expand(*first.shape, 1, hd)
    return [torch.where(ok, torch.gather(x, -2, at).squeeze(-2), 0.0) for x in _values(tiles, hd)]


# --- inputs ---------------------------------------------------------------------------------------
def _filled(c, gen, n_page):
    """A cache whose pages hold quantised noise, some dimensions wider than others as keys have them."""
    nkv, hd = HEADS[c["heads"]][1:]
    nb = _blocks(hd)
    cache = torch.zeros(n_page, nkv, c["page"] // TILE * 576 * nb, dtype=torch.uint8, device="cuda")
    wide = torch.exp(0.5 * torch.randn(2, nkv, hd, device="cuda", generator=gen))
    each = max(1, (1 << 25) // (nkv * c["page"] * hd))
    ident = dict(c)
    for at in range(0, n_page, each):
        n = min(each, n_page - at)
        kv = torch.randn(2, n, c["page"], nkv, hd, device="cuda", generator=gen) * wide[:, None, None]
        pages = torch.arange(at, at + n, device="cuda")[:, None]
        pos = torch.arange(c["page"], device="cuda").expand(n, c["page"])
        _store(ident, cache, pages, pos, torch.ones_like(pos, dtype=torch.bool), kv[0], kv[1])
    return cache


def _spoil(c, cache, table, lens):
    """What lies past each sequence's length in its last page, and in the pages that belong to nobody: scales that are NaN."""
    hd = HEADS[c["heads"]][2]
    tiles = cache.view(cache.shape[0], cache.shape[1], c["page"] // TILE, -1)
    used = torch.zeros(cache.shape[0], c["page"], dtype=torch.bool)
    for row, n in zip(table, lens):
        for i in range(-(-n // c["page"])):
            used[row[i], :min(c["page"], n - i * c["page"])] = True
    bad = (~used).reshape(-1, c["page"] // TILE, TILE).cuda()[:, None, :, :, None]
    nb = _blocks(hd)
    codes, scales = TILE * 16 * nb, TILE * 2 * nb
    for at in (codes, 2 * codes + scales):
        part = tiles[..., at:at + scales].reshape(*tiles.shape[:3], TILE, 2 * nb)
        tiles[..., at:at + scales] = part.masked_fill(bad, 255).reshape(*tiles.shape[:3], scales)


def _settings(c, gen):
    """Temperature, top-k, top-p and min-p of every row."""
    n = c["rows"]
    kinds = {"none": [0], "k": [1], "p": [2], "min": [3], "all": [4], "mixed": [0, 1, 2, 3, 4, 5]}[c["filters"]]
    kind = torch.tensor([kinds[i % len(kinds)] for i in range(n)], device="cuda")
    rand = torch.rand(4, n, device="cuda", generator=gen)
    temp = torch.where(kind == 5, 0.0, 0.6 + 0.7 * rand[0])
    k = torch.where((kind == 1) | (kind == 4), 2 + (98 * rand[1]), 0.0).int()
    p = torch.where((kind == 2) | (kind == 4), 0.8 + 0.19 * rand[2], 1.0)
    low = torch.where((kind == 3) | (kind == 4), 0.01 + 0.09 * rand[3], 0.0)
    return temp, k, p, low


def _logits(c, gen):
    """A step's logits: noise with a head of likely tokens, one token in a hundred barred."""
    n, V = c["rows"], c["vocab"]
    x = torch.randn(n, V, device="cuda", generator=gen) * 2
    at = torch.randint(0, V, (n, 64), device="cuda", generator=gen)
    x.scatter_add_(1, at, 6 - 4 * torch.log(torch.rand(n, 64, device="cuda", generator=gen).clamp_min(1e-6)))
    x.masked_fill_(torch.rand(n, V, device="cuda", generator=gen) < 0.01, -math.inf)
    return x.to(DTYPES[c["dtype"]])


def _undecided(x, u, temp, k, p, low):
    """Rows where a limit falls nearer to a border than 32 bits tell apart."""
    s, _ = torch.sort(x.double(), dim=1, descending=True, stable=True)
    y = (s - s[:, :1]) / temp.double().clamp_min(1e-3)[:, None]
    w = torch.exp(y)
    rank = torch.arange(x.shape[1], device=x.device)
    w = torch.where((k[:, None] > 0) & (rank >= k[:, None]), 0.0, w)
    cum = torch.cumsum(w, 1)
    total = cum[:, -1:]
    before = cum - w
    near = (((before - p.double()[:, None] * total).abs() < 1e-6 * total) & (p < 1)[:, None]).any(1)
    near |= (((y - torch.log(low.double()).clamp_min(-1e3)[:, None]).abs() < 1e-5) & (low > 0)[:, None]).any(1)
    keep = ((before < p.double()[:, None] * total) | (p >= 1)[:, None]) & (w > 0) & (y >= torch.log(low.double())[:, None])
    keep[:, 0] = True
    kept = torch.where(keep, w, 0.0).sum(1, keepdim=True)
    near |= (((cum - u.double()[:, None] * kept).abs() < 1e-6 * kept) & keep).any(1)
    return near & (temp > 0)


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    if c["op"] == "sample":
        n = c["rows"]
        x, u = _logits(c, gen), torch.rand(n, device="cuda", generator=gen)
        st = _settings(c, gen)
        for _ in range(40):
            bad = _undecided(x, u, *st)
            if not bool(bad.any()):
                break
            u = torch.where(bad, torch.rand(n, device="cuda", generator=gen), u)
            st = tuple(torch.where(bad, b, a) for a, b in zip(st, _settings(c, gen)))
        return {"case": c, "logits": x, "u": u, "temperature": st[0], "top_k": st[1], "top_p": st[2], "min_p": st[3],
                "token": torch.empty(n, dtype=torch.int32, device="cuda"), "logprob": torch.empty(n, device="cuda")}
    nh, nkv, hd = HEADS[c["heads"]]
    n, nq = c["seqs"], c["queries"]
    (lens, new), (table, n_page) = _lengths(c), _pages(c)
    st = {"case": c, "pages": torch.tensor(table, dtype=torch.int32, device="cuda"),
          "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
          "new": torch.tensor(new, dtype=torch.int32, device="cuda"),
          "q": (1.5 * torch.randn(n, nq, nh, hd, device="cuda", generator=gen)).to(dt),
          "out": torch.zeros(n, nq, nh, hd, dtype=dt, device="cuda")}
    st["cache"] = _filled(c, gen, n_page)
    _spoil(c, st["cache"], table, lens)
    if c["op"] == "attention":
        st["lse"] = torch.zeros(n, nq, nh, device="cuda")
        return st
    wide = torch.exp(0.5 * torch.randn(2, 1, 1, nkv, hd, device="cuda", generator=gen))
    kv = torch.randn(2, n, nq, nkv, hd, device="cuda", generator=gen) * wide
    st["k"], st["v"] = kv[0].to(dt), kv[1].to(dt)
    angle = torch.arange(c["length"], device="cuda").double()[:, None] / 500000.0 ** (torch.arange(hd // 2, device="cuda") * 2 / hd)
    st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
    st["start"] = st["lens"] - st["new"]
    return st


# --- one pass ---------------------------------------------------------------------------------------
def _rotated(x, cos, sin, halves):
    """x [seqs, n, heads, hd] turned by cos and sin [seqs, n, hd/2], in 64 bits."""
    hd = x.shape[-1]
    x, cos, sin = x.double(), cos.double()[:, :, None], sin.double()[:, :, None]
    a, b = (x[..., :hd // 2], x[..., hd // 2:]) if halves else (x[..., 0::2], x[..., 1::2])
    a, b = a * cos - b * sin, a * sin + b * cos
    return torch.cat([a, b], -1) if halves else torch.stack([a, b], -1).flatten(-2)


def _plain_append(c, st):
    hd = HEADS[c["heads"]][2]
    t = torch.arange(c["queries"], device="cuda")
    ok = t < st["new"][:, None]
    pos = torch.where(ok, st["start"][:, None] + t, 0).long()
    cos, sin = st["cos"][pos], st["sin"][pos]
    q = _rotated(st["q"], cos, sin, c["halves"]).to(st["q"].dtype)
    q = torch.where(ok[..., None, None], q, st["out"])
    k = _rotated(st["k"], cos, sin, c["halves"]).float()
    _store(c, st["cache"], st["pages"], pos, ok, k, st["v"].float())
    k, v = _load(c, st["cache"], st["pages"], st["start"], c["queries"], st["lens"])
    return {"q": q, "k": k.to(st["q"].dtype), "v": v.to(st["q"].dtype)}


def _plain_attention(c, q, cache, pages, lens):
    nh, nkv, hd = HEADS[c["heads"]]
    n, nq, gq = c["seqs"], c["queries"], nh // nkv
    tiles = cache.view(cache.shape[0], nkv, c["page"] // TILE, -1)[pages.long()]       # seqs pages heads tiles bytes
    k, v = (x.transpose(1, 2).reshape(n, nkv, -1, hd) for x in _values(tiles, hd))     # seqs heads positions hd
    at = torch.arange(k.shape[2], device=q.device)
    held = (at < lens[:, None])[:, None, :, None]
    k, v = torch.where(held, k, 0.0), torch.where(held, v, 0.0)
    x = q.float().reshape(n, nq, nkv, gq, hd).permute(0, 2, 1, 3, 4) * (1 / math.sqrt(hd))
    s = torch.matmul(x.reshape(n, nkv, nq * gq, hd), k.transpose(2, 3)).reshape(n, nkv, nq, gq, -1)
    seen = at < (lens[:, None] - (nq - 1 - torch.arange(nq, device=q.device)))[..., None]   # seqs nq positions
    s = s.masked_fill(~seen[:, None, :, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e.reshape(n, nkv, nq * gq, -1), v).reshape(n, nkv, nq, gq, hd) / total
    lse = (top + torch.log(total)).squeeze(-1)
    return {"out": out.permute(0, 2, 1, 3, 4).reshape(n, nq, nh, hd).to(q.dtype),
            "lse": lse.permute(0, 2, 1, 3).reshape(n, nq, nh)}


def _plain_sample(x, u, temp, k, p, low):
    s, at = torch.sort(x.float(), dim=1, descending=True, stable=True)
    greedy = temp <= 0
    y = (s - s[:, :1]).double() / torch.where(greedy, 1.0, temp).double()[:, None]
    rank = torch.arange(s.shape[1], device=s.device)
    w = torch.exp(y)
    w = torch.where((k[:, None] > 0) & (rank >= k[:, None]), 0.0, w)
    cum = torch.cumsum(w, 1)
    keep = ((cum - w < p.double()[:, None] * cum[:, -1:]) | (p >= 1)[:, None]) & (w >= low.double()[:, None])
    keep = torch.where(greedy[:, None], rank == 0, keep | (rank == 0))
    w = torch.where(keep, w, 0.0)
    cum = torch.cumsum(w, 1)
    total = cum[:, -1:]
    pick = ((cum <= u.double()[:, None] * total) & (rank < keep.sum(1, keepdim=True) - 1)).sum(1, keepdim=True)
    return {"token": torch.gather(at, 1, pick)[:, 0].int(), "logprob": torch.log(torch.gather(w, 1, pick) / total)[:, 0].float()}


def run(state):
    c = state["case"]
    if c["op"] == "sample":
        args = [state[k] for k in ("logits", "u", "temperature", "top_k", "top_p", "min_p")]
        if not own:
            return _plain_sample(*args)
        if "sample" not in state:
            state["sample"] = _fwb()[1].sample_rows
        state["sample"](args[0], args[1], temperature=args[2], top_k=args[3], top_p=args[4], min_p=args[5],
                        token=state["token"], logprob=state["logprob"])
        return {"token": state["token"], "logprob": state["logprob"]}
    if c["op"] == "append":
        if not own:
            return _plain_append(c, state)
        if "kv4" not in state:
            state["kv4"] = _fwb()[0]
        kv4 = state["kv4"]
        kv4.append(state["q"], state["k"], state["v"], state["cache"], state["pages"], state["lens"], cos=state["cos"],
                   sin=state["sin"], halves=c["halves"], n_new=state["new"], q_out=state["out"])
        k, v = kv4.read(state["cache"], state["pages"], state["start"], c["queries"], head_dim=HEADS[c["heads"]][2],
                        dtype=DTYPES[c["dtype"]], lengths=state["lens"])
        return {"q": state["out"], "k": k, "v": v}
    if not own:
        return _plain_attention(c, state["q"], state["cache"], state["pages"], state["lens"])
    if "plan" not in state:
        nh, nkv, hd = HEADS[c["heads"]]
        state["plan"] = _fwb()[0].Attention(n_seq=c["seqs"], n_query=c["queries"], n_head=nh, n_head_kv=nkv, head_dim=hd,
                                            dtype=DTYPES[c["dtype"]], page_size=c["page"], n_page=state["cache"].shape[0],
                                            max_pages=state["pages"].shape[1])
    state["plan"](state["q"], state["cache"], state["pages"], state["lens"], out=state["out"], lse=state["lse"])
    return {"out": state["out"], "lse": state["lse"]}


# --- from the definition, in 64 bits -------------------------------------------------------------------
def _rows64(cache, pages, n, hd):
    """Keys and values [heads, n, hd] in 64 bits of the first n positions on these pages: each code looked up by where the
    format puts it."""
    nb, nkv, dev = _blocks(hd), cache.shape[1], cache.device
    t = cache[pages].reshape(len(pages), nkv, -1, 576 * nb).transpose(0, 1).reshape(nkv, -1, 576 * nb)
    nibs = torch.stack([t & 15, t >> 4], -1).flatten(-2)
    got = []
    for value in (False, True):
        at = torch.empty(TILE, hd, dtype=torch.long)
        for p in range(TILE):
            for i in range(hd):
                b, r = divmod(i, 32)
                if value:
                    at[p, i] = 576 * nb + 2 * (p * 16 * nb + ((r // 4) ^ (4 if p % 4 >= 2 else 0)) * 2 * nb + 2 * b) + r % 4
                else:
                    at[p, i] = 2 * (p * 16 * nb + r // 8 * 4 * nb + 4 * b) + r % 8 // 2 + 4 * (r % 2)
        code = nibs[..., at.to(dev)].flatten(1, 2)[:, :n].double() - 8
        first = (288 * nb if value else 0) + 256 * nb
        d = t[..., first:first + 32 * nb].contiguous().view(torch.float16).reshape(nkv, -1, nb)[:, :n].double()
        got.append(code * d[..., torch.arange(hd, device=dev) // 32])
    return got


def exact(case, seed):
    c = case
    st = prepare(c, seed)
    if c["op"] == "sample":
        x, u = st["logits"].double(), st["u"].double()
        tokens, logp = [], []
        for i in range(c["rows"]):
            t, k, p, low = (float(st[name][i]) for name in ("temperature", "top_k", "top_p", "min_p"))
            if t <= 0:
                tokens.append(int(x[i].argmax()))
                logp.append(0.0)
                continue
            order = torch.argsort(x[i], descending=True, stable=True)
            prob = torch.softmax(x[i] / t, 0)[order]
            if k > 0:
                prob = prob[:int(k)]
            keep = len(prob)
            if p < 1:
                keep = int((torch.cumsum(prob, 0) < p * prob.sum()).sum()) + 1
            prob = prob[:max(1, min(keep, int((prob >= low * prob[0]).sum())))]
            at = min(int((torch.cumsum(prob, 0) <= u[i] * prob.sum()).sum()), len(prob) - 1)
            tokens.append(int(order[at]))
            logp.append(float(torch.log(prob[at] / prob.sum())))
        return {"token": torch.tensor(tokens, dtype=torch.int32), "logprob": torch.tensor(logp, dtype=torch.float64)}
    nh, nkv, hd = HEADS[c["heads"]]
    (lens, new), nq = _lengths(c), c["queries"]
    if c["op"] == "append":
        got = {"q": torch.zeros(*st["q"].shape, dtype=torch.float64, device="cuda")}
        half = torch.arange(hd // 2, device="cuda")
        one, other = (half, half + hd // 2) if c["halves"] else (2 * half, 2 * half + 1)
        for name in ("q", "k", "v"):
            out = torch.zeros(*st[name].shape, dtype=torch.float64, device="cuda")
            for s in range(c["seqs"]):
                x = st[name][s, :new[s]].double()
                if name != "v":
                    at = slice(lens[s] - new[s], lens[s])
                    z = torch.complex(x[..., one], x[..., other]) * torch.complex(st["cos"][at].double(), st["sin"][at].double())[:, None]
                    x = torch.empty_like(x)
                    x[..., one], x[..., other] = z.real, z.imag
                if name != "q":   # from the nearest fp32 value, in blocks of 32
                    x = x.float().double()
                    for b in range(0, hd, 32):
                        y = x[..., b:b + 32]
                        far = y.abs().amax(-1, keepdim=True)
                        d = (torch.where((y == far).any(-1, keepdim=True), -far, far) / 8).half().double()
                        x[..., b:b + 32] = (torch.floor(y / d + 0.5).clamp(-8, 7) * d).nan_to_num(0.0)
                out[s, :new[s]] = x
            got[name] = out
        return got
    out = torch.zeros(c["seqs"], nq, nh, hd, dtype=torch.float64, device="cuda")
    lse = torch.zeros(c["seqs"], nq, nh, dtype=torch.float64, device="cuda")
    for s in range(c["seqs"]):
        n = lens[s]
        k, v = _rows64(st["cache"], st["pages"][s, :-(-n // c["page"])].long(), n, hd)
        for h in range(nkv):
            q = st["q"][s, :, h * (nh // nkv):(h + 1) * (nh // nkv)].double()          # nq gq hd
            a = torch.einsum("qgd,td->gqt", q, k[h]) / math.sqrt(hd)
            a.masked_fill_(torch.arange(n, device="cuda") >= (n - nq + 1 + torch.arange(nq, device="cuda"))[:, None], -math.inf)
            lse[s, :, h * (nh // nkv):(h + 1) * (nh // nkv)] = a.logsumexp(2).transpose(0, 1)
            out[s, :, h * (nh // nkv):(h + 1) * (nh // nkv)] = torch.einsum("gqt,td->qgd", a.softmax(2), v[h])
    return {"out": out, "lse": lse}
