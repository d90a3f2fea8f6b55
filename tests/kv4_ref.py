"""The 4-bit cache's operators from their definitions, in 64 bits (CPU or GPU tensors)."""
import math

import torch

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def turned(x, cos, sin, halves):
    """x [..., tokens, heads, hd] by cos and sin [..., tokens, hd/2], in 64 bits."""
    hd = x.shape[-1]
    x, cos, sin = x.double(), cos.double().unsqueeze(-2), sin.double().unsqueeze(-2)
    one, other = (x[..., :hd // 2], x[..., hd // 2:]) if halves else (x[..., ::2], x[..., 1::2])
    out = torch.empty_like(x)
    a, b = one * cos - other * sin, one * sin + other * cos
    if halves:
        out[..., :hd // 2], out[..., hd // 2:] = a, b
    else:
        out[..., ::2], out[..., 1::2] = a, b
    return out


def held(y):
    """What blocks of 32 of the fp32 values y [..., hd] come back as, in 64 bits."""
    y = y.float().double()
    out = torch.empty_like(y)
    for b in range(0, y.shape[-1], 32):
        z = y[..., b:b + 32]
        hi, lo = z.amax(-1, keepdim=True).clamp_min(0), z.amin(-1, keepdim=True).clamp_max(0)
        m = torch.where(hi >= -lo, hi, lo)
        d = (m / -8).clamp(-65504, 65504).float().half().double()
        code = torch.where(d == 0, 0.0, torch.floor(z / d + 0.5).clamp(-8, 7))
        w = code * d
        w[(~torch.isfinite(z)).any(-1, keepdim=True).expand(w.shape)] = math.nan
        out[..., b:b + 32] = w
    return out


class Pages:
    """Pages of a cache for sequences of these lengths, scattered; the rest of the cache holds 0xff (NaN scales)."""

    def __init__(self, kv4, lengths, heads, hd, page, seed=0, spare=3, room=0, fill=0xff):
        need = [-(-(n + room) // page) for n in lengths]
        self.n_page = sum(need) + spare
        gen = torch.Generator().manual_seed(seed)
        order = torch.randperm(self.n_page, generator=gen).tolist()
        wide = max(max(need), 1)
        table = torch.full((len(lengths), wide), -1, dtype=torch.int32)
        for s, n in enumerate(need):
            for i in range(n):
                table[s, i] = order.pop()
        self.page, self.hd, self.heads = page, hd, heads
        self.table = table.cuda()
        self.cache = kv4.empty(self.n_page, heads, hd, page).fill_(fill)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")


def filled(kv4, lengths, heads, hd, page, seed=0, scale=1.0, **kw):
    """Pages with noise in all positions below the lengths -> (Pages, k, v), k and v what read() gives for every
    sequence, fp32 [n_seq, longest, heads, hd]."""
    p = Pages(kv4, lengths, heads, hd, page, seed, **kw)
    n, most = len(lengths), max(max(lengths), 1)
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    kv = torch.randn(2, n, most, heads, hd, device="cuda", generator=gen) * scale
    new = p.lengths.clone()
    kv4.append(None, kv[0], kv[1], p.cache, p.table, p.lengths, n_new=new)
    k, v = kv4.read(p.cache, p.table, torch.zeros_like(p.lengths), most, head_dim=hd, dtype=torch.float32, lengths=p.lengths)
    return p, k, v


def attention(q, k, v, lengths, n_new=None, scale=None):
    """(out, lse, mass, reach) in 64 bits of q [n_seq, n_query, n_head, hd] over k, v [n_seq, most, heads, hd]; mass: the
    same average of |v|, reach: the largest scale * sum |q||k| of a row. NaN rows where a token has no row."""
    n, nq, nh, hd = q.shape
    heads = k.shape[2]
    scale = scale or 1 / math.sqrt(hd)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mass, lse = out.clone(), torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=q.device)
    reach = torch.zeros_like(lse)
    for s in range(n):
        fresh = nq if n_new is None else int(n_new[s])
        for t in range(fresh):
            m = int(lengths[s]) - (fresh - 1 - t)
            if m <= 0:
                continue
            x = q[s, t].double().reshape(heads, nh // heads, hd)
            kk, vv = k[s, :m].double(), v[s, :m].double()
            a = torch.einsum("hgd,thd->hgt", x, kk) * scale
            w = a.softmax(-1)
            out[s, t] = torch.einsum("hgt,thd->hgd", w, vv).reshape(nh, hd)
            mass[s, t] = torch.einsum("hgt,thd->hgd", w, vv.abs()).reshape(nh, hd)
            lse[s, t] = a.logsumexp(-1).flatten()
            reach[s, t] = (torch.einsum("hgd,thd->hgt", x.abs(), kk.abs()) * scale).amax(-1).flatten()
    return out, lse, mass, reach


def bounds(q, out, lse, mass, reach, most, heads):
    """How far a call's out and lse may be from these. Scores: a product of 32 exact pairs is summed in fp32 whose
    additions may truncate (2^-23 each, 32 + 4 + 2 of them, queries of fp32 calls held to 2^-22): under 2^-17 of reach.
    The average: twice the scores' errors, probabilities with their scales held to 2^-11 (fp32 calls 2^-21) and exp2 to
    2^-21, sums of `most` terms in fp32;
    and the output's rounding. bf16 calls of many rows hold keys and values to 2^-11 as well. Products below 2^-24 of 2^8 times the largest scale are lost: 2^-20 of mass's largest covers them."""
    p = 2.0 ** -11 if q.dtype != torch.float32 else 2.0 ** -21
    ds = 2.0 ** -17 * reach
    if q.dtype == torch.bfloat16 and q.shape[1] * (q.shape[2] // heads) >= 64:
        ds, p = ds + 2.0 ** -11 * reach, p + 2.0 ** -11
    rel = p + 2.0 ** -20 + 2 * ds + (most / 16 + 32) * 2.0 ** -23
    tol = mass * rel[..., None] + mass.amax(-1, keepdim=True) * 2.0 ** -20 + out.abs() * half_step(q.dtype)
    return tol, ds + 2.0 ** -20 + lse.abs() * 2.0 ** -23


def check_attention(got, got_lse, q, k, v, lengths, n_new=None, scale=None):
    out, lse, mass, reach = attention(q, k, v, lengths, n_new, scale)
    tol, tol_lse = bounds(q, out, lse.nan_to_num(neginf=0.0), mass, reach, k.shape[1], k.shape[2])
    for s in range(q.shape[0]):
        fresh = q.shape[1] if n_new is None else int(n_new[s])
        d = (got[s, :fresh].double() - out[s, :fresh]).abs()
        assert bool((d <= tol[s, :fresh]).all()), (s, float((d / tol[s, :fresh].clamp_min(1e-300)).max()))
        a, b = got_lse[s, :fresh].double(), lse[s, :fresh]
        empty = torch.isinf(b)
        assert torch.equal(torch.isinf(a), empty)
        d = torch.where(empty, 0.0, (a - b).abs().nan_to_num(nan=math.inf, posinf=math.inf) if not bool(empty.any()) else
                        torch.where(empty, 0.0, a - b).abs())
        assert bool((d <= tol_lse[s, :fresh]).all()), (s, float(d.max()))
