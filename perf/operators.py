"""Beam search next to the decode path: what its operators compute, and on which sizes they are timed.

Three operators (fwb.beam), in a plain form written with elementary torch operations and as the library's kernels:

- attention of a batch of sequences that share a prefix: each group of beams attends to one copy of its prompt's keys and
  values and to the positions that its own sequence has added (the suffix), with one softmax over both;
- the selection of a beam step: the best n_select of beams x vocabulary by accumulated log-probability;
- the reordering of per-beam state (token and slot tables, key/value rows) by the parents that the selection chose.

Lengths and ancestries follow from the case alone, so that `work` counts what a pass needs; values follow from the seed.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i32": torch.int32}
ESIZE = {"f32": 4, "f16": 2, "bf16": 2, "i32": 4}
HEADS = {"8b": (32, 8, 128), "70b": (64, 8, 128), "small": (4, 2, 128), "tp8": (8, 8, 128), "tiny": (6, 6, 48)}


def _beam():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "forword.c_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from fwb import beam
    return beam


def _attn(name, dtype, heads, groups, beams, queries, prefix, suffix, slots):
    return {"name": name, "op": "attention", "dtype": dtype, "heads": heads, "groups": groups, "beams": beams,
            "queries": queries, "prefix": prefix, "suffix": suffix, "slots": slots}


def _select(name, dtype, groups, beams, vocab, select):
    return {"name": name, "op": "select", "dtype": dtype, "groups": groups, "beams": beams, "vocab": vocab, "select": select}


def _reorder(name, dtype, outer, groups, beams, inner, cap, used, width, in_place):
    return {"name": name, "op": "reorder", "dtype": dtype, "outer": outer, "groups": groups, "beams": beams, "inner": inner,
            "cap": cap, "used": used, "width": width, "in_place": in_place}


def listed():
    return [
        # one layer of the first steps of a beam search after a short question, on the 8B model's fp32 cache: latency
        _attn("attn_f32_short", "f32", "8b", 1, 4, 1, 200, 9, True),
        # the same late in a long context (8000 positions of the 8192)
        _attn("attn_f32_long", "f32", "8b", 1, 4, 1, 8000, 64, True),
        # the small model's six 48-wide heads, three beams, odd lengths
        _attn("attn_f32_tiny", "f32", "tiny", 1, 3, 1, 251, 33, True),
        # eight beams on a long document kept in fp16
        _attn("attn_f16_beams", "f16", "8b", 1, 8, 1, 8191, 160, True),
        # a server's batch: six prompts of different lengths, five beams each
        _attn("attn_f16_groups", "f16", "8b", 6, 5, 1, 6001, 100, True),
        # checking seven drafted tokens for each of nine continuations of one prompt
        _attn("attn_bf16_drafts", "bf16", "8b", 1, 9, 7, 4099, 71, False),
        # 64 samples of one long prompt on the 70B shape, ragged continuations
        _attn("attn_bf16_samples", "bf16", "70b", 1, 64, 1, 32763, 512, False),
        # the step of a four-beam search on the small model's vocabulary: latency
        _select("select_f32_step", "f32", 1, 4, 32000, 8),
        # sixteen beams on the large vocabulary, logits in bf16 (many equal ones)
        _select("select_bf16_wide", "bf16", 1, 16, 128256, 32),
        # a server's batch of 32 searches
        _select("select_f32_batch", "f32", 32, 8, 128256, 16),
        # the slot table of a four-beam search
        _reorder("reorder_table", "i32", 1, 1, 4, 1, 256, 131, 1, True),
        # 100 of 128 continued positions of K and V of all 32 layers, moved in place
        _reorder("reorder_cache", "f32", 64, 1, 8, 8, 128, 100, 128, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "select", "reorder"])
    if op == "attention":
        largest = _work(listed()[6])
        while True:
            c = _attn("", rng.choice(["f32", "f16", "bf16"]), rng.choice(sorted(HEADS)), _log(rng, 1, 8), _log(rng, 1, 64),
                      rng.choice([1, 1, 1, _log(rng, 2, 8)]), _log(rng, 16, 32768), 0, rng.random() < 0.5)
            c["suffix"] = c["queries"] + _log(rng, 1, 512) - 1
            w = _work(c)
            rate = 10 if c["dtype"] == "f32" else 1   # fp32 products run at a tenth of the tensor rate
            if w["flops"] * rate <= largest["flops"] and w["bytes"] <= largest["bytes"]:
                break
    elif op == "select":
        while True:
            c = _select("", rng.choice(["f32", "f16", "bf16"]), _log(rng, 1, 64), _log(rng, 1, 32), _log(rng, 1000, 128256), 0)
            c["select"] = c["beams"] * rng.choice([1, 2])
            if c["groups"] * c["beams"] * c["vocab"] <= 32 * 8 * 128256:
                break
    else:
        while True:
            kind = rng.choice(["i32", "f32", "f16"])
            c = _reorder("", kind, 1, _log(rng, 1, 8), _log(rng, 2, 32), 1, _log(rng, 16, 512), 0, 1, rng.random() < 0.5)
            if kind != "i32":
                c["outer"], c["inner"], c["width"] = 2 * _log(rng, 2, 32), rng.choice([2, 6, 8]), rng.choice([48, 64, 128])
            c["used"] = rng.randint(max(1, c["cap"] // 8), c["cap"])
            if c["outer"] * c["groups"] * c["beams"] * c["inner"] * c["cap"] * c["width"] * ESIZE[kind] <= 64 * 8 * 8 * 128 * 128 * 4:
                break
    del c["name"]
    return c


# --- lengths and ancestries: from the case alone -------------------------------------------------
def _lengths(c):
    """(prefix length of each group, suffix length of each sequence): the first is full, the others shorter."""
    p = [max(1, c["prefix"] - (g * c["prefix"] * 2) // (3 * c["groups"])) for g in range(c["groups"])]
    room = c["suffix"] - c["queries"]
    n = c["groups"] * c["beams"]
    if c["slots"]:   # beams of one search are equally long
        s = [c["suffix"] - (g * room) // (2 * c["groups"]) for g in range(c["groups"]) for _ in range(c["beams"])]
    else:            # samples end where they end
        s = [c["suffix"] - (i * 37 % n) * room // n for i in range(n)]
    return p, s


def _ancestry(c):
    """slots[sequence][position] = the beam slot (within the group) whose cache row holds it, as a search leaves it behind:
    the newest positions are a beam's own, older ones come from its ancestors."""
    rng = np.random.default_rng([c["groups"], c["beams"], c["suffix"]])
    own_slot = np.arange(c["beams"], dtype=np.int32)
    table = np.zeros((c["groups"], c["beams"], c["suffix"]), np.int32)
    for rows in table:
        for t in range(c["suffix"]):
            parents = np.sort(np.where(rng.random(c["beams"]) < 0.4, rng.integers(0, c["beams"], c["beams"]), own_slot))
            rows[:] = rows[parents]
            rows[:, t] = own_slot
    return table.reshape(-1, c["suffix"])


def _parents(c):
    """Each group's parents. In place a pass is repeated on its own result, so a survivor keeps its slot there."""
    rng = random.Random("%d %d %d" % (c["groups"], c["beams"], c["used"]))
    table = []
    for _ in range(c["groups"]):
        n = c["beams"]
        if c["in_place"]:
            live = sorted(rng.sample(range(n), max(1, (n + 1) // 2)))
            table.append([b if b in live else rng.choice(live) for b in range(n)])
        else:
            table.append([rng.randrange(n) for _ in range(n)])
    return table


def _work(c):
    if c["op"] == "attention":
        nh, nkv, hd = HEADS[c["heads"]]
        e = ESIZE[c["dtype"]]
        p, s = _lengths(c)
        nq = c["queries"]
        rows = c["groups"] * c["beams"] * nq * nh
        if c["slots"]:
            table = _ancestry(c)
            held = 0
            for g in range(c["groups"]):   # the beams of a group are equally long
                held_by = np.sort(table[g * c["beams"]:(g + 1) * c["beams"], :s[g * c["beams"]]], axis=0)
                held += held_by.shape[1] + int((held_by[1:] != held_by[:-1]).sum())
        else:
            held = sum(s)
        kv = (sum(p) + held) * nkv * hd * 2 * e
        pairs = sum(c["beams"] * nq * n for n in p) + sum(nq * n - nq * (nq - 1) // 2 for n in s)
        return {"bytes": kv + 2 * rows * hd * e + rows * 4, "flops": 4 * pairs * nh * hd}
    if c["op"] == "select":
        n = c["groups"] * c["beams"]
        return {"bytes": n * c["vocab"] * ESIZE[c["dtype"]] + n * 4 + c["groups"] * c["select"] * 12, "flops": 4 * n * c["vocab"]}
    run = c["used"] * c["width"] * ESIZE[c["dtype"]]
    moved = 0
    for par in _parents(c):
        into = [b for b in range(c["beams"]) if not c["in_place"] or par[b] != b]
        moved += len(into) + len({par[b] for b in into})
    return {"bytes": c["outer"] * c["inner"] * run * moved + c["groups"] * c["beams"] * 4, "flops": 0}


def work(case):
    return _work(case)


# --- inputs ---------------------------------------------------------------------------------------
def _select_inputs(c, gen):
    """A step's logits: noise with a head of likely tokens, one token in a hundred barred; and the beams' scores so far."""
    G, W, V = c["groups"], c["beams"], c["vocab"]
    x = torch.randn(G, W, V, device="cuda", generator=gen) * 2
    at = torch.randint(0, V, (G, W, 64), device="cuda", generator=gen)
    up = 6 - 4 * torch.log(torch.rand(G, W, 64, device="cuda", generator=gen).clamp_min(1e-6))
    x.scatter_add_(2, at, up)
    x.masked_fill_(torch.rand(G, W, V, device="cuda", generator=gen) < 0.01, -math.inf)
    scores = -8 * torch.rand(G, W, device="cuda", generator=gen)
    return x.to(DTYPES[c["dtype"]]), scores


def _undecided(c, x, scores):
    """Groups in which two neighbours among the best are nearer than rounding can tell apart; equal logits of one row are a
    tie that the lower index wins, and stay."""
    x = x.float()
    s = (x - torch.logsumexp(x, 2, keepdim=True) + scores[:, :, None]).flatten(1)
    top, at = s.topk(min(c["select"] + 4, s.shape[1]), dim=1)
    near = (top[:, :-1] - top[:, 1:]) < 2e-5
    row = at // c["vocab"]
    lx = x.flatten(1).gather(1, at)
    tie = (row[:, :-1] == row[:, 1:]) & (lx[:, :-1] == lx[:, 1:])
    return (near & ~tie).any(1)


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if c["op"] == "attention":
        nh, nkv, hd = HEADS[c["heads"]]
        n, dt = c["groups"] * c["beams"], DTYPES[c["dtype"]]

        def rand(*shape, sd=1.0):
            return (torch.randn(*shape, device="cuda", generator=gen) * sd).to(dt)

        p, s = _lengths(c)
        st = {"case": c, "q": rand(n, c["queries"], nh, hd, sd=1.5),
              "pk": rand(c["groups"], nkv, c["prefix"], hd), "pv": rand(c["groups"], nkv, c["prefix"], hd),
              "sk": rand(n, nkv, c["suffix"], hd), "sv": rand(n, nkv, c["suffix"], hd),
              "plen": torch.tensor(p, dtype=torch.int32, device="cuda"),
              "slen": torch.tensor(s, dtype=torch.int32, device="cuda"),
              "slots": torch.from_numpy(_ancestry(c)).cuda() if c["slots"] else None,
              "out": torch.empty(n, c["queries"], nh, hd, dtype=dt, device="cuda"),
              "lse": torch.empty(n, c["queries"], nh, device="cuda")}
        # past a group's or a sequence's length the cache holds whatever was there before
        at = torch.arange(c["prefix"], device="cuda")
        for name in ("pk", "pv"):
            st[name].masked_fill_((at >= st["plen"][:, None])[:, None, :, None], math.nan)
        return st
    if c["op"] == "select":
        x, scores = _select_inputs(c, gen)
        for _ in range(20):
            bad = _undecided(c, x, scores)
            if not bool(bad.any()):
                break
            y, t = _select_inputs(c, gen)
            x = torch.where(bad[:, None, None], y, x)
            scores = torch.where(bad[:, None], t, scores)
        k = (c["groups"], c["select"])
        return {"case": c, "logits": x, "scores": scores, "out": torch.empty(k, device="cuda"),
                "parent": torch.empty(k, dtype=torch.int32, device="cuda"),
                "token": torch.empty(k, dtype=torch.int32, device="cuda")}
    shape = (c["outer"], c["groups"] * c["beams"], c["inner"], c["cap"], c["width"])
    if c["dtype"] == "i32":
        src = torch.randint(0, 128256, shape, dtype=torch.int32, device="cuda", generator=gen)
    else:
        src = torch.randn(shape, device="cuda", generator=gen).to(DTYPES[c["dtype"]])
    return {"case": c, "src": src, "dst": src if c["in_place"] else torch.zeros_like(src),
            "parent": torch.tensor(_parents(c), dtype=torch.int32, device="cuda")}


# --- one pass ---------------------------------------------------------------------------------------
def _plain_attention(c, q, pk, pv, sk, sv, plen, slen, slots):
    G, W, nq = c["groups"], c["beams"], c["queries"]
    nh, nkv, hd = HEADS[c["heads"]]
    gq, P, S = nh // nkv, c["prefix"], c["suffix"]
    dt = q.dtype
    dev = q.device
    q = q.float().reshape(G, W, nq, nkv, gq, hd).permute(0, 3, 1, 2, 4, 5) * (1 / math.sqrt(hd))   # G kv W nq gq hd
    held = (torch.arange(P, device=dev) < plen[:, None])[:, None, :]                               # G 1 P
    pk = torch.where(held[..., None], pk, torch.zeros((), dtype=dt, device=dev)).float()
    pv = torch.where(held[..., None], pv, torch.zeros((), dtype=dt, device=dev)).float()
    ps = torch.matmul(q.reshape(G, nkv, W * nq * gq, hd), pk.transpose(2, 3))                      # G kv rows P
    ps = ps.masked_fill(~held[:, :, None], -math.inf).reshape(G, nkv, W, nq, gq, P)
    at = torch.arange(S, device=dev)
    if slots is not None:
        seq = (slots.long().reshape(G, W, S) + W * torch.arange(G, device=dev)[:, None, None])
        sk, sv = sk[seq, :, at].permute(0, 3, 1, 2, 4), sv[seq, :, at].permute(0, 3, 1, 2, 4)      # G kv W S hd
    else:
        sk, sv = (t.reshape(G, W, nkv, S, hd).transpose(1, 2) for t in (sk, sv))
    sk, sv = sk.float(), sv.float()
    ss = torch.matmul(q.reshape(G, nkv, W, nq * gq, hd), sk.transpose(3, 4)).reshape(G, nkv, W, nq, gq, S)
    seen = at < (slen.reshape(G, W, 1, 1) - (nq - 1 - torch.arange(nq, device=dev))[:, None])       # G W nq S
    ss = ss.masked_fill(~seen[:, None, :, :, None], -math.inf)
    top = torch.maximum(ps.amax(-1), ss.amax(-1))[..., None]
    ep, es = torch.exp(ps - top), torch.exp(ss - top)
    total = (ep.sum(-1) + es.sum(-1))[..., None]
    out = torch.matmul(ep.reshape(G, nkv, W * nq * gq, P), pv).reshape(G, nkv, W, nq, gq, hd)
    out = out + torch.matmul(es.reshape(G, nkv, W, nq * gq, S), sv).reshape(G, nkv, W, nq, gq, hd)
    out = (out / total).permute(0, 2, 3, 1, 4, 5).reshape(G * W, nq, nh, hd)
    lse = (top + torch.log(total))[..., 0].permute(0, 2, 3, 1, 4).reshape(G * W, nq, nh)
    return out.to(dt), lse


def _plain_select(c, logits, scores):
    x = logits.float()
    top = x.amax(2, keepdim=True)
    logp = (x - top) - torch.log(torch.exp(x - top).sum(2, keepdim=True))
    s, at = torch.sort((logp + scores[:, :, None]).flatten(1), dim=1, descending=True, stable=True)
    s, at = s[:, :c["select"]], at[:, :c["select"]]
    return s, (at // c["vocab"]).int(), (at % c["vocab"]).int()


def run(state):
    c = state["case"]
    if c["op"] == "attention":
        if not own:
            out, lse = _plain_attention(c, *(state[k] for k in ("q", "pk", "pv", "sk", "sv", "plen", "slen", "slots")))
            return {"out": out, "lse": lse}
        if "plan" not in state:
            nh, nkv, hd = HEADS[c["heads"]]
            state["plan"] = _beam().PrefixAttention(n_group=c["groups"], n_beam=c["beams"], n_query=c["queries"], n_head=nh,
                                                    n_head_kv=nkv, head_dim=hd, dtype=DTYPES[c["dtype"]],
                                                    prefix_cap=c["prefix"], suffix_cap=c["suffix"])
        state["plan"](state["q"], state["pk"], state["pv"], state["sk"], state["sv"], prefix_len=state["plen"],
                      suffix_len=state["slen"], slots=state["slots"], out=state["out"], lse=state["lse"])
        return {"out": state["out"], "lse": state["lse"]}
    if c["op"] == "select":
        if not own:
            s, parent, token = _plain_select(c, state["logits"], state["scores"])
            return {"scores": s, "parent": parent, "token": token}
        if "plan" not in state:
            state["plan"] = _beam().BeamSelect(n_group=c["groups"], n_beam=c["beams"], n_vocab=c["vocab"],
                                               n_select=c["select"], dtype=DTYPES[c["dtype"]])
        state["plan"](state["logits"], state["scores"], out_scores=state["out"], parent=state["parent"], token=state["token"])
        return {"scores": state["out"], "parent": state["parent"], "token": state["token"]}
    src, dst, used = state["src"], state["dst"], c["used"]
    if own:
        if "reorder" not in state:
            state["reorder"] = _beam().reorder
        # the positions in use of every slot, moved as a view of the whole state
        state["reorder"](src[:, :, :, :used], state["parent"], dst[:, :, :, :used])
        return dst
    par = state["parent"].long() + c["beams"] * torch.arange(c["groups"], device="cuda")[:, None]
    dst[:, :, :, :used] = src[:, par.flatten(), :, :used]
    return dst


# --- from the definition, in 64 bits -------------------------------------------------------------------
def exact(case, seed):
    c = case
    st = prepare(c, seed)
    if c["op"] == "reorder":
        want = (st["dst"] if not c["in_place"] else st["src"]).double()
        for g, par in enumerate(_parents(c)):
            for b, p in enumerate(par):
                want[:, g * c["beams"] + b, :, :c["used"]] = st["src"][:, g * c["beams"] + p, :, :c["used"]].double()
        return want if c["dtype"] != "i32" else None
    if c["op"] == "select":
        best = []
        for g in range(c["groups"]):
            x = st["logits"][g].double()
            best.append((x.log_softmax(1) + st["scores"][g].double()[:, None]).flatten().topk(c["select"]).values)
        return {"scores": torch.stack(best), "parent": None, "token": None}
    nh, nkv, hd = HEADS[c["heads"]]
    p, s = _lengths(c)
    n, nq = c["groups"] * c["beams"], c["queries"]
    table = torch.from_numpy(_ancestry(c)).long().cuda() if c["slots"] else None
    out = torch.zeros(n, nq, nh, hd, dtype=torch.float64, device="cuda")
    lse = torch.zeros(n, nq, nh, dtype=torch.float64, device="cuda")
    for g in range(c["groups"]):
        gk, gv = (st[k][g, :, :p[g]].double() for k in ("pk", "pv"))
        for i in range(g * c["beams"], (g + 1) * c["beams"]):
            if table is not None:
                at = torch.arange(s[i], device="cuda")
                src = table[i, :s[i]] + g * c["beams"]
                k, v = (st[k][src, :, at].transpose(0, 1).double() for k in ("sk", "sv"))
            else:
                k, v = (st[k][i, :, :s[i]].double() for k in ("sk", "sv"))
            k, v = torch.cat([gk, k], 1), torch.cat([gv, v], 1)
            for t in range(nq):
                m = p[g] + s[i] - (nq - 1 - t)
                a = torch.einsum("hgd,htd->hgt", st["q"][i, t].double().reshape(nkv, nh // nkv, hd), k[:, :m]) / math.sqrt(hd)
                out[i, t] = torch.einsum("hgt,htd->hgd", a.softmax(2), v[:, :m]).reshape(nh, hd)
                lse[i, t] = a.logsumexp(2).flatten()
    return {"out": out, "lse": lse}
