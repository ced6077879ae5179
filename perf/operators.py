"""The cache operators and the sizes they are measured at.

Three operators serve the tokens that come after a long prefill: attention of a
batch's new tokens over a prefix that its sequences share and over their own
caches, the attention weight that each cached key has received, and the
eviction of the keys that received least.  ``run`` computes them in their plain
form, or with the package's operators where ``own`` is true; ``exact`` computes
them from their definitions in 64 bits.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

# Elements of one block of plain-form scores (fp32), to bound its memory.
_BLOCK = 1 << 27


def _ops():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "minference-npu_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from minference import ops

    return ops


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
# op       shared: attention over a shared prefix and own caches
#          weights: attention weight per cached key
#          evict: eviction by weight
# B, Hq, Hkv, D     sequences, query heads, key/value heads, head dim
# Sq       new tokens per sequence; C own cache capacity; P prefix length;
# G        prefixes (each shared by B / G sequences)
# ragged   own lengths differ (and end before the capacity)
# layout   "bhsd" caches are contiguous; "bshd" caches keep a token's heads together
# lse      the log-sum-exp is returned (shared) or known from the attention (weights)


def _shared(name, B, Hq, Hkv, D, Sq, P, C, dtype="bf16", G=1, ragged=True, layout="bhsd",
            lse=False):
    return dict(name=name, op="shared", B=B, Hq=Hq, Hkv=Hkv, D=D, Sq=Sq, P=P, C=C, G=G,
                dtype=dtype, ragged=ragged, layout=layout, lse=lse)


def _weights(name, B, Hq, Hkv, D, Sq, C, dtype="bf16", ragged=False, layout="bhsd", lse=False):
    return dict(name=name, op="weights", B=B, Hq=Hq, Hkv=Hkv, D=D, Sq=Sq, C=C, dtype=dtype,
                ragged=ragged, layout=layout, lse=lse)


def _evict(name, B, Hkv, D, C, keep, sink, recent, dtype="bf16", ragged=False, layout="bhsd"):
    return dict(name=name, op="evict", B=B, Hkv=Hkv, D=D, C=C, keep=keep, sink=sink,
                recent=recent, dtype=dtype, ragged=ragged, layout=layout)


def listed():
    return [
        # a few short chats over one system prompt: the latency of a decode step
        _shared("shared_step_short", 4, 32, 32, 96, 1, 1024, 256),
        # a batch of questions decoding over one 64K document, grouped heads
        _shared("shared_step_grouped", 32, 32, 8, 128, 1, 65536, 512),
        # the same with one key/value head per query head and token-major caches
        _shared("shared_step_heads", 16, 32, 32, 96, 1, 16383, 1024, dtype="fp16",
                layout="bshd", lse=True),
        # five drafted tokens per sequence, two documents, few key/value heads
        _shared("shared_drafts", 24, 32, 4, 64, 5, 8191, 700, G=2, lse=True),
        # questions of 128 tokens entering a 16K document at once
        _shared("shared_questions", 8, 32, 8, 128, 128, 16384, 384),
        # no prefix: a decode step over two long caches
        _shared("cache_step_long", 2, 32, 32, 96, 1, 0, 65536, lse=True),
        # the weights of one decode step, added to those of the steps before
        _weights("weights_step", 16, 32, 8, 128, 1, 8192, ragged=True, lse=True),
        # the weights of a 64K prompt's last 64 queries
        _weights("weights_window", 1, 32, 32, 96, 64, 65536),
        # the weights of every query of a 16K prompt
        _weights("weights_prefill", 1, 32, 32, 96, 16384, 16384, dtype="fp16"),
        # four short caches halved
        _evict("evict_short", 4, 8, 64, 1025, 512, 4, 64),
        # a 64K prompt's cache cut to an eighth after its prefill
        _evict("evict_long", 1, 32, 96, 65536, 8192, 4, 64),
        # a serving batch that reached its budget, token-major caches
        _evict("evict_batch", 32, 8, 128, 4097, 2048, 4, 256, dtype="fp16", ragged=True,
               layout="bshd"),
    ]


_MAX_FLOPS = 8.2e11
_MAX_BYTES = 1.6e9


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _draw_once(rng):
    op = rng.choice(["shared", "shared", "weights", "evict"])
    D = rng.choice([64, 80, 96, 128])
    common = dict(dtype=rng.choice(["bf16", "fp16"]), ragged=rng.random() < 0.6,
                  layout=rng.choice(["bhsd", "bshd"]))
    Hkv = rng.choice([2, 4, 8, 16, 32])
    group = rng.choice([1, 1, 2, 4, 7, 8])
    if op == "shared":
        G = rng.choice([1, 1, 1, 2, 3])
        B = G * _log_int(rng, 1, 48 // G)
        Sq = rng.choice([1, 1, 1, _log_int(rng, 2, 8), _log_int(rng, 9, 160)])
        P = rng.choice([0, 1, 1, 1]) * _log_int(rng, 16, 65536)
        C = Sq + _log_int(rng, 1, 65536 if P == 0 else 2048)
        return _shared("", B, Hkv * group, Hkv, D, Sq, P, C, G=G, lse=rng.random() < 0.5, **common)
    if op == "weights":
        B = _log_int(rng, 1, 32)
        C = _log_int(rng, 64, 65536)
        Sq = min(C, rng.choice([1, 1, _log_int(rng, 2, 64), 64, C]))
        return _weights("", B, Hkv * group, Hkv, D, Sq, C, lse=rng.random() < 0.5, **common)
    B = _log_int(rng, 1, 32)
    C = _log_int(rng, 64, 65536)
    keep = max(8, int(C * rng.choice([0.125, 0.25, 0.5, 0.8])))
    sink = rng.choice([0, 4, 4, 8])
    return _evict("", B, Hkv, D, C, keep, sink, rng.randint(0, keep - sink), **common)


def draw(rng):
    while True:
        case = _draw_once(rng)
        del case["name"]
        cost = work(case)
        if (cost["flops"] <= _MAX_FLOPS and cost["bytes"] <= _MAX_BYTES
                and case["B"] * case["Hkv"] * case["C"] * case["D"] <= 2 * 32 * 65536 * 96):
            return case


def _lengths(case, cap, n):
    """Valid rows of n caches of `cap` rows: whole, or spread between half and all
    with one that holds the new tokens only.  The seed shuffles them."""
    if not case["ragged"]:
        return [cap] * n
    out = [cap - (i * cap) // (2 * n) for i in range(n)]
    if n >= 4:
        out[-1] = min(cap, case.get("Sq", 1))
    return out


def _pairs(case, lens):
    """(row, key) pairs of the own caches that a causal row sees, per query head."""
    Sq = case["Sq"]
    total = 0
    for n in lens:
        first = n - Sq + 1  # keys that row 0 sees
        lo = max(first, 0)
        rows = n - lo + 1
        total += (lo + n) * rows // 2
    return total


def work(case):
    B, Hkv, D, C = case["B"], case["Hkv"], case["D"], case["C"]
    lens = _lengths(case, C, B)
    own_rows = Hkv * sum(lens)
    if case["op"] == "evict":
        kept = Hkv * sum(min(n, case["keep"]) for n in lens)
        return {"bytes": 4 * own_rows + kept * (2 * 2 * 2 * D + 8), "flops": 0}
    Hq, Sq = case["Hq"], case["Sq"]
    rows = B * Hq * Sq
    if case["op"] == "weights":
        return {"bytes": 2 * D * (rows + own_rows) + 8 * Hkv * B * C
                + (4 * rows if case["lse"] else 0),
                "flops": 2 * D * Hq * _pairs(case, lens)}
    plens = _prefix_lengths(case)
    return {"bytes": 2 * D * (2 * rows + 2 * own_rows + 2 * Hkv * sum(plens)),
            "flops": 4 * D * (Hq * _pairs(case, lens) + Hq * Sq * (B // case["G"]) * sum(plens))}


def _prefix_lengths(case):
    return [case["P"] - (i * case["P"]) // (2 * case["G"]) for i in range(case["G"])]


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _cache(g, B, H, S, D, dtype, layout, sinks):
    """A cache of keys or values [B,H,S,D]; `sinks` positions of every head are
    scaled up, the columns that a long prompt's queries attend to."""
    shape = (B, S, H, D) if layout == "bshd" else (B, H, S, D)
    x = torch.empty(shape, dtype=dtype, device="cuda")
    x.normal_(generator=g)
    if layout == "bshd":
        x = x.transpose(1, 2)
    if sinks and S:
        pos = torch.randint(0, S, (min(sinks, S),), generator=g, device="cuda")
        x[:, :, pos] = x[:, :, pos] * 4
    return x


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = {"bf16": torch.bfloat16, "fp16": torch.float16}[case["dtype"]]
    B, Hkv, D, C = case["B"], case["Hkv"], case["D"], case["C"]
    perm = torch.randperm(B, generator=torch.Generator().manual_seed(seed))
    lens = torch.tensor(_lengths(case, C, B), dtype=torch.int32)[perm].cuda()
    st = dict(case=case, lengths=lens if case["ragged"] else None)
    if case["op"] == "evict":
        st["k"] = _cache(g, B, Hkv, C, D, dtype, case["layout"], 32)
        st["v"] = _cache(g, B, Hkv, C, D, dtype, case["layout"], 0)
        # heavy-tailed weights, some of them exactly zero (underflowed): ties
        w = torch.randn(B, Hkv, C, generator=g, device="cuda").mul_(2).exp_()
        w *= torch.rand(B, Hkv, C, generator=g, device="cuda") > 0.3
        st["weights"] = w
        return st
    Hq, Sq = case["Hq"], case["Sq"]
    q = torch.empty(B, Sq, Hq, D, dtype=dtype, device="cuda").normal_(generator=g)
    st["q"] = q.transpose(1, 2)  # a projection's rows: token-major
    st["k"] = _cache(g, B, Hkv, C, D, dtype, case["layout"], 32 if C >= 1024 else 1)
    if case["op"] == "weights":
        st["weights"] = torch.rand(B, Hkv, C, generator=g, device="cuda")
        st["out"] = torch.empty_like(st["weights"])
        if case["lse"]:
            st["lse"] = torch.empty(B, Hq, Sq, device="cuda")
            grouped = st["lse"].unflatten(1, (Hkv, Hq // Hkv))
            for b, heads, rows in _blocks(st):
                s = _own_scores(st, b, heads, rows).double()
                grouped[b, heads, :, rows] = torch.logsumexp(s, -1).float()
        return st
    st["v"] = _cache(g, B, Hkv, C, D, dtype, case["layout"], 0)
    st["kp"] = st["vp"] = st["prefix_lengths"] = None
    if case["P"]:
        G, P = case["G"], case["P"]
        st["kp"] = _cache(g, G, Hkv, P, D, dtype, case["layout"], 32)
        st["vp"] = _cache(g, G, Hkv, P, D, dtype, case["layout"], 0)
        if G > 1:
            st["prefix_lengths"] = torch.tensor(_prefix_lengths(case), dtype=torch.int32).cuda()
    return st


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------


def _blocks(st):
    """(sequence, kv heads, rows): blocks of queries whose scores fit _BLOCK elements."""
    c = st["case"]
    per_row = (c["Hq"] // c["Hkv"]) * max(c["C"], 1)
    rows = max(1, min(c["Sq"], _BLOCK // per_row))
    heads = max(1, min(c["Hkv"], _BLOCK // (per_row * rows)))
    for b in range(c["B"]):
        for h in range(0, c["Hkv"], heads):
            for r in range(0, c["Sq"], rows):
                yield b, slice(h, min(c["Hkv"], h + heads)), slice(r, min(c["Sq"], r + rows))


def _own_scores(st, b, heads, rows):
    """Scaled scores [kv heads, group, rows, C] of one sequence, -inf where hidden."""
    c = st["case"]
    q = st["q"][b].unflatten(0, (c["Hkv"], c["Hq"] // c["Hkv"]))[heads, :, rows].float()
    k = st["k"][b, heads].float()
    s = torch.matmul(q, k.transpose(1, 2)[:, None]) / math.sqrt(c["D"])
    n = c["C"] if st["lengths"] is None else st["lengths"][b]
    r = torch.arange(rows.start, rows.stop, device="cuda")[:, None]
    return s.masked_fill(torch.arange(c["C"], device="cuda") >= n - (c["Sq"] - 1 - r),
                         float("-inf"))


def _plain_shared(st):
    c = st["case"]
    B, Hq, Hkv, D, Sq, P, C, G = (c[x] for x in ("B", "Hq", "Hkv", "D", "Sq", "P", "C", "G"))
    group, n = Hq // Hkv, B // G
    scale = 1.0 / math.sqrt(D)
    out = torch.empty(B, Hkv, group, Sq, D, dtype=st["q"].dtype, device="cuda")
    lse = torch.empty(B, Hkv, group, Sq, device="cuda")
    query = st["q"].unflatten(1, (Hkv, group))
    cols = torch.arange(C, device="cuda")
    rows = torch.arange(Sq, device="cuda")
    lens = st["lengths"]
    if lens is None:
        lens = torch.full((B,), C, dtype=torch.int32, device="cuda")
    hidden = cols >= (lens[:, None] - (Sq - 1 - rows))[:, :, None]  # [B, Sq, C]
    stale = cols >= lens[:, None]  # rows past a length hold anything
    step = max(1, min(Hkv, _BLOCK // (n * group * Sq * (P + C))))
    for g in range(G):
        sl = slice(g * n, (g + 1) * n)
        for h in range(0, Hkv, step):
            hs = slice(h, min(Hkv, h + step))
            q = query[sl, hs].float()  # [n, heads, group, Sq, D]
            s_own = torch.matmul(q, st["k"][sl, hs].float().transpose(2, 3)[:, :, None]) * scale
            s_own = s_own.masked_fill(hidden[sl][:, None, None], float("-inf"))
            m = s_own.amax(-1, keepdim=True)
            if P:
                # every sequence's rows against the prefix in one product
                flat = q.transpose(0, 1).reshape(q.shape[1], -1, D)
                s_pre = torch.matmul(flat, st["kp"][g, hs].float().transpose(1, 2)) * scale
                if st["prefix_lengths"] is not None:
                    past = torch.arange(P, device="cuda") >= st["prefix_lengths"][g]
                    s_pre = s_pre.masked_fill(past, float("-inf"))
                m_pre = s_pre.amax(-1).view(-1, n, group, Sq).transpose(0, 1)
                m = torch.maximum(m, m_pre[..., None])
            m0 = m.clamp_min(-3e38)
            p = torch.exp(s_own - m0)
            l = p.sum(-1, keepdim=True)
            v = st["v"][sl, hs].float().masked_fill(stale[sl][:, None, :, None], 0.0)
            o = torch.matmul(p, v[:, :, None])
            if P:
                p = torch.exp(s_pre - m0.transpose(0, 1).reshape(q.shape[1], -1, 1))
                l = l + p.sum(-1).view(-1, n, group, Sq).transpose(0, 1)[..., None]
                o_pre = torch.matmul(p, st["vp"][g, hs].float())
                o = o + o_pre.view(-1, n, group, Sq, D).transpose(0, 1)
            out[sl, hs] = torch.where(l > 0, o / l, torch.zeros_like(o)).to(out.dtype)
            lse[sl, hs] = (m + torch.log(l))[..., 0]
    out = out.flatten(1, 2)
    return {"out": out, "lse": lse.flatten(1, 2)} if c["lse"] else {"out": out}


def _plain_weights(st):
    c = st["case"]
    acc = st["weights"].double()
    for b, heads, rows in _blocks(st):
        s = _own_scores(st, b, heads, rows)
        if c["lse"]:
            lse = st["lse"][b].unflatten(0, (c["Hkv"], -1))[heads, :, rows, None]
            lse = lse.clamp_min(-3e38)  # a row that sees nothing adds nothing
        else:
            m = s.amax(-1, keepdim=True).clamp_min(-3e38)
            lse = m + torch.log(torch.exp(s - m).sum(-1, keepdim=True)).clamp_min(0.0)
        acc[b, heads] += torch.exp(s - lse).sum((1, 2), dtype=torch.float64)
    return {"weights": acc.float()}


def _plain_evict(st):
    c = st["case"]
    B, Hkv, D, C, keep = (c[x] for x in ("B", "Hkv", "D", "C", "keep"))
    lens = st["lengths"]
    if lens is None:
        lens = torch.full((B,), C, dtype=torch.int32, device="cuda")
    n = lens.view(B, 1, 1)
    j = torch.arange(C, device="cuda")
    forced = (j < c["sink"]) | (j >= n - c["recent"])
    score = st["weights"].masked_fill(forced, float("inf")).masked_fill(j >= n, float("-inf"))
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :keep]
    slot = torch.arange(keep, device="cuda")
    index = order.masked_fill(slot >= n, C).sort(-1).values
    kept = index < C
    index = torch.where(kept, index, -1)
    src = index.clamp_min(0)
    rows = src[..., None].expand(-1, -1, -1, D)
    return {
        "k": torch.gather(st["k"], 2, rows).masked_fill(~kept[..., None], 0.0),
        "v": torch.gather(st["v"], 2, rows).masked_fill(~kept[..., None], 0.0),
        "weights": torch.gather(st["weights"], 2, src).masked_fill(~kept, 0.0),
        "index": index.int(),
        "lengths": lens.clamp_max(keep),
    }


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def run(state):
    c = state["case"]
    if not own:
        return {"shared": _plain_shared, "weights": _plain_weights,
                "evict": _plain_evict}[c["op"]](state)
    ops = _ops()
    if c["op"] == "shared":
        res = ops.shared_prefix_attention(
            state["q"], state["kp"], state["vp"], state["k"], state["v"], state["lengths"],
            prefix_lengths=state["prefix_lengths"], return_lse=c["lse"])
        return {"out": res[0], "lse": res[1]} if c["lse"] else {"out": res}
    if c["op"] == "weights":
        return {"weights": ops.accumulate_attention_weights(
            state["q"], state["k"], state["weights"], state["lengths"], lse=state.get("lse"),
            out=state["out"])}
    res = ops.evict_cache(state["k"], state["v"], state["weights"], c["keep"], state["lengths"],
                          sink=c["sink"], recent=c["recent"])
    return {"k": res.k, "v": res.v, "weights": res.weights, "index": res.index,
            "lengths": res.lengths}


# ---------------------------------------------------------------------------
# Definitions in 64 bits
# ---------------------------------------------------------------------------


def _exact_rows(c, st, b, head):
    """Per block of query rows of one head: (first row, its scores in natural
    logarithms over [prefix, own keys], values over the same keys)."""
    h = head // (c["Hq"] // c["Hkv"])
    n = c["C"] if st["lengths"] is None else int(st["lengths"][b])
    keys = [st["k"][b, h, :n].double()]
    vals = [st["v"][b, h, :n].double()] if "v" in st else []
    P = 0
    if st.get("kp") is not None:
        g = b // (c["B"] // c["G"])
        P = c["P"] if st["prefix_lengths"] is None else int(st["prefix_lengths"][g])
        keys.insert(0, st["kp"][g, h, :P].double())
        vals.insert(0, st["vp"][g, h, :P].double())
    keys = torch.cat(keys)
    vals = torch.cat(vals) if vals else None
    q = st["q"][b, head].double() * c["D"] ** -0.5
    step = max(1, (1 << 26) // max(1, keys.shape[0]))
    for r0 in range(0, c["Sq"], step):
        s = q[r0:r0 + step] @ keys.T
        row = torch.arange(r0, r0 + s.shape[0], device=s.device).unsqueeze(1)
        col = torch.arange(keys.shape[0], device=s.device).unsqueeze(0)
        hidden = col - P > n - c["Sq"] + row
        yield r0, torch.where(hidden, -math.inf, s), vals


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "evict":
        return _exact_evict(case, st)
    B, Hq, Sq = case["B"], case["Hq"], case["Sq"]
    if case["op"] == "weights":
        acc = st["weights"].double()
        group = Hq // case["Hkv"]
        for b in range(B):
            for head in range(Hq):
                for r0, s, _ in _exact_rows(case, st, b, head):
                    if case["lse"]:
                        z = st["lse"][b, head, r0:r0 + s.shape[0]].double()
                    else:
                        z = torch.logsumexp(s, 1)
                    p = torch.exp(s - torch.where(torch.isinf(z), 0.0, z)[:, None])
                    acc[b, head // group, :s.shape[1]] += p.sum(0)
        return {"weights": acc}
    out = torch.zeros(B, Hq, Sq, case["D"], dtype=torch.float64, device="cuda")
    lse = torch.zeros(B, Hq, Sq, dtype=torch.float64, device="cuda")
    for b in range(B):
        for head in range(Hq):
            for r0, s, vals in _exact_rows(case, st, b, head):
                z = torch.logsumexp(s, 1)
                lse[b, head, r0:r0 + s.shape[0]] = z
                p = torch.exp(s - torch.where(torch.isinf(z), 0.0, z)[:, None])
                out[b, head, r0:r0 + s.shape[0]] = p @ vals
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


def _exact_evict(c, st):
    B, H, C, keep = c["B"], c["Hkv"], c["C"], c["keep"]
    w = st["weights"].cpu().numpy().astype(np.float64)
    lens = [C] * B if st["lengths"] is None else st["lengths"].tolist()
    index = np.full((B, H, keep), -1, dtype=np.int64)
    for b, n in enumerate(lens):
        head = set(range(min(c["sink"], n))) | set(range(max(0, n - c["recent"]), n))
        must = np.array(sorted(head), dtype=np.int64)
        free = np.setdiff1d(np.arange(n), must)
        room = min(n, keep) - len(must)
        for h in range(H):
            by_weight = free[np.lexsort((free, -w[b, h, free]))]
            picked = np.sort(np.concatenate([must, by_weight[:max(0, room)]]))
            index[b, h, :len(picked)] = picked
    at = torch.from_numpy(index).cuda()
    live = (at >= 0).double()
    bi = torch.arange(B, device="cuda")[:, None, None]
    hi = torch.arange(H, device="cuda")[None, :, None]
    at0 = at.clamp(min=0)
    return {
        "k": st["k"][bi, hi, at0].double() * live[..., None],
        "v": st["v"][bi, hi, at0].double() * live[..., None],
        "weights": st["weights"][bi, hi, at0].double() * live,
        "index": at,
        "lengths": torch.tensor([min(n, keep) for n in lens], device="cuda"),
    }
