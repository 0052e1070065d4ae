"""Workloads of the decode step's operators: a MoE layer for a few tokens, and a bounded latent cache (the attention
weight every cached row has received, and the eviction of the rows that received least).

`listed()` and `draw()` describe cases, `prepare()` makes their inputs on the GPU, `run()` is one pass - through the
library's operators when `own` is true, through elementary torch operations in 32 bits otherwise - and `exact()` the
same result from the definition in 64 bits.  `work()` counts the bytes and operations a pass cannot do without.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

PAGE = 64


# ------------------------------------------------------------------------------------------------------------------ cases
def _moe(name, T, d, f, E, k, shared):
    return {"name": name, "op": "moe_few", "T": T, "d": d, "f": f, "E": E, "k": k, "shared": shared}


def _acc(name, B, H, Sq, lo, hi, d=576, page=PAGE, dtype="bf16"):
    return {"name": name, "op": "accumulate", "B": B, "H": H, "Sq": Sq, "len_lo": lo, "len_hi": hi, "d": d, "page": page,
            "dtype": dtype}


def _evict(name, B, lo, hi, keep, recent, d=576, page=PAGE, dtype="bf16"):
    return {"name": name, "op": "evict", "B": B, "len_lo": lo, "len_hi": hi, "keep": keep, "recent": recent, "d": d,
            "page": page, "dtype": dtype}


def listed():
    return [
        # one token through a small layer: nothing but latency
        _moe("moe_t1_small", 1, 1024, 512, 8, 2, False),
        # one token of a single user through the layer the benchmark times at 4096 tokens
        _moe("moe_t1_d4096", 1, 4096, 1024, 64, 8, True),
        # one token through a layer of the model-wide widths (7168, 256 experts, top-8): eight experts and the shared one
        _moe("moe_t1_d7168", 1, 7168, 2048, 256, 8, True),
        # an odd batch and widths that are multiples of 64 only
        _moe("moe_t37_odd", 37, 2112, 704, 40, 5, False),
        # a full decode batch: nearly every expert is read for four tokens
        _moe("moe_t128_d7168", 128, 7168, 2048, 256, 8, True),
        # one short sequence of a small rank (heads split over GPUs)
        _acc("acc_b1_h16", 1, 16, 1, 900, 900),
        # the decode configuration: 128 sequences of 4096 keys, 128 heads
        _acc("acc_b128_h128", 128, 128, 1, 4096, 4096),
        # the last 32 queries of long prompts of different lengths (an observation window after prefill)
        _acc("acc_window32", 2, 128, 32, 5000, 16384),
        # fp32 cache, narrow rows, short pages
        _acc("acc_fp32_d160", 2, 8, 1, 100, 3000, d=160, page=16, dtype="fp32"),
        # one sequence a few rows over its bound
        _evict("evict_b1_small", 1, 1061, 1061, 1000, 64),
        # a batch cut to half
        _evict("evict_b128_half", 128, 4096, 4096, 2048, 128),
        # few long sequences of different lengths cut to one bound; shorter ones stay as they are
        _evict("evict_long_ragged", 8, 16384, 131072, 32768, 512),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["moe_few", "accumulate", "evict"])
    if op == "moe_few":
        while True:
            E = _logint(rng, 4, 256)
            c = _moe(None, _logint(rng, 1, 128), 64 * _logint(rng, 4, 112), 64 * _logint(rng, 2, 32), E,
                     rng.randint(1, min(8, E)), rng.random() < 0.5)
            if 6 * c["E"] * c["d"] * c["f"] <= 6_000_000_000:
                break
    elif op == "accumulate":
        if rng.random() < 0.25:                                       # the kernels for other types and widths
            c = _acc(None, rng.randint(1, 4), rng.randint(1, 16), rng.choice([1, 1, 3]), 1, _logint(rng, 8, 3000),
                     d=8 * rng.randint(2, 40), page=rng.choice([1, 16, 48, 64]), dtype=rng.choice(["bf16", "fp32"]))
        else:
            Sq = rng.choice([1, 1, 1, _logint(rng, 2, 32)])
            B = _logint(rng, 1, 64 if Sq == 1 else 3)
            hi = _logint(rng, 4, 16384 if Sq == 1 else 8192)
            c = _acc(None, B, rng.choice([1, 8, 16, 37, 64, 128, 128]), Sq, max(1, hi // rng.choice([1, 2, 50])), hi,
                     d=rng.choice([64, 192, 576, 576]), page=rng.choice([64, 128]))
    else:
        B = _logint(rng, 1, 64)
        hi = _logint(rng, 4, min(131072, 400_000 // B))
        keep = max(1, int(hi * rng.uniform(0.1, 1.0)))
        c = _evict(None, B, max(1, hi // rng.choice([1, 2, 20])), hi, keep, int(keep * rng.choice([0.0, 0.02, 0.3, 1.0])),
                   d=rng.choice([64, 160, 576, 576]), page=rng.choice([16, 64, 64]), dtype=rng.choice(["bf16", "bf16", "fp32"]))
    del c["name"]
    return c


def _lengths(case):
    """Sequence lengths of a case: spread evenly from the longest down to the shortest, fixed by the case alone."""
    B, lo, hi = case["B"], case["len_lo"], case["len_hi"]
    return [hi if B == 1 else hi - (hi - lo) * i // (B - 1) for i in range(B)]


def work(case):
    if case["op"] == "moe_few":
        T, d, f, E, k = (case[n] for n in ("T", "d", "f", "E", "k"))
        # experts that T tokens with k choices each are expected to touch when the choices are uniform
        active = E * (1.0 - (1.0 - k / E) ** T) + (1 if case["shared"] else 0)
        rows = T * k + (T if case["shared"] else 0)
        return {"bytes": int(active * 3 * d * f * 2 + 4 * d * E + 4 * T * d),
                "flops": int(rows * 6 * d * f + 2 * T * d * E)}
    es = 4 if case["dtype"] == "fp32" else 2
    lens, d = _lengths(case), case["d"]
    if case["op"] == "accumulate":
        H, Sq = case["H"], case["Sq"]
        pairs = sum(max(0, n + i + 1 - Sq) for n in lens for i in range(Sq)) * H
        return {"bytes": sum(lens) * (d * es + 8) + len(lens) * H * Sq * (d * es + 8), "flops": 2 * pairs * d}
    moves = 0.0
    for n in lens:
        K, R = min(case["keep"], n), min(case["recent"], n)
        moves += min(R, n - K) + (max(0, n - K - R) * (K - R) / (n - R) if n > R else 0)
    return {"bytes": int(sum(lens) * 8 + sum(min(case["keep"], n) for n in lens) * 4 + moves * (2 * d * es + 16)), "flops": 0}


# ----------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _prepare_moe(case, seed):
    g = _gen(seed)
    T, d, f, E = (case[n] for n in ("T", "d", "f", "E"))

    def w(*shape, fan_in):
        return torch.empty(*shape, dtype=torch.bfloat16, device="cuda").normal_(0.0, 1.0 / math.sqrt(fan_in), generator=g)
    st = {"case": case, "x": w(T, d, fan_in=1.0),
          "Wg": torch.empty(d, E, device="cuda").normal_(0.0, 1.0 / math.sqrt(d), generator=g),
          "W1": w(E, d, f, fan_in=d), "W3": w(E, d, f, fan_in=d), "W2": w(E, f, d, fan_in=f), "shared": None}
    if case["shared"]:
        st["shared"] = (w(d, f, fan_in=d), w(d, f, fan_in=d), w(f, d, fan_in=f))
    return st


def _tables(case, g):
    """A pool with the case's sequences on randomly permuted pages; a few pages belong to nobody."""
    lens, page = _lengths(case), case["page"]
    per = [(n + page - 1) // page for n in lens]
    num_pages = sum(per) + 3
    perm = torch.randperm(num_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(per), dtype=torch.int32, device="cuda")
    o = 0
    for b, k in enumerate(per):
        table[b, :k] = perm[o:o + k]
        o += k
    return lens, num_pages, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


def _rows(table_row, n, page):
    """Physical row of every logical row 0 .. n-1 of a sequence."""
    t = torch.arange(n, device=table_row.device)
    return table_row.long()[t // page] * page + t % page


def _visible(n, Sq, H, device):
    """[H * Sq, n] mask of the keys each query sees: the last query sees all n keys (bottom-right alignment)."""
    i = torch.arange(Sq, device=device).repeat(H)
    return torch.arange(n, device=device)[None, :] <= (i + n - Sq)[:, None]


def _prepare_accumulate(case, seed):
    g = _gen(seed)
    dt = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
    lens, num_pages, table, seqlens = _tables(case, g)
    B, H, Sq, d, page = (case[n] for n in ("B", "H", "Sq", "d", "page"))
    pool = torch.empty(num_pages, page, d, dtype=dt, device="cuda").normal_(generator=g)
    Q = torch.empty(B, H, Sq, d, dtype=dt, device="cuda").normal_(generator=g)
    # weights received so far
    weights = torch.empty(num_pages, page, device="cuda").normal_(generator=g).exp_()
    scale = 1.0 / math.sqrt(d)
    # the row statistics that the attention of the same step returned
    m = torch.empty(B, H, Sq, device="cuda")
    l = torch.empty(B, H, Sq, device="cuda")
    flat = pool.view(-1, d)
    for b, n in enumerate(lens):
        keys = flat[_rows(table[b], n, page)].float()
        q = Q[b].reshape(H * Sq, d).float()
        step = max(1, (1 << 27) // n)                                  # queries at a time: half a GB of scores
        vis = None if Sq == 1 else _visible(n, Sq, H, "cuda")
        mm, ll = [], []
        for r in range(0, H * Sq, step):
            s = q[r:r + step] @ keys.T * scale
            if vis is not None:
                s.masked_fill_(~vis[r:r + step], float("-inf"))
            mx = s.max(dim=1).values
            e = torch.exp(s - torch.where(torch.isinf(mx), torch.zeros_like(mx), mx)[:, None])
            mm.append(mx)
            ll.append(e.sum(dim=1))
        m[b], l[b] = torch.cat(mm).view(H, Sq), torch.cat(ll).view(H, Sq)
    if Sq == 1:
        Q, m, l = Q[:, :, 0].contiguous(), m[:, :, 0].contiguous(), l[:, :, 0].contiguous()
    return {"case": case, "Q": Q, "pool": pool, "table": table, "seqlens": seqlens, "lens": lens, "m": m, "l": l,
            "weights": weights, "scale": scale}


def _prepare_evict(case, seed):
    g = _gen(seed)
    dt = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
    lens, num_pages, table, seqlens = _tables(case, g)
    d, page = case["d"], case["page"]
    pool = torch.empty(num_pages, page, d, dtype=dt, device="cuda").normal_(generator=g)
    # few rows hold most of the weight; one row in ten has received none (ties)
    weights = torch.empty(num_pages * page, device="cuda").normal_(0.0, 2.0, generator=g).exp_()
    weights *= torch.rand(num_pages * page, device="cuda", generator=g) > 0.1
    # every sequence has been cut before: an eighth of the positions are missing and the rows are not in order, but the
    # newest ones still are at the end
    positions = torch.full((num_pages * page,), -1, dtype=torch.int32, device="cuda")
    nxt = []
    for b, n in enumerate(lens):
        seen = n + n // 8
        tail = min(case["recent"], n)
        older = torch.randperm(seen - tail, generator=g, device="cuda")[: n - tail]
        p = torch.cat((older, torch.arange(seen - tail, seen, device="cuda")))
        positions[_rows(table[b], n, page)] = p.to(torch.int32)
        nxt.append(seen)
    # (sequence, new row) of every row that survives: known on the host, which knows the lengths
    K = [min(case["keep"], n) for n in lens]
    flat_b = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(K)).cuda()
    flat_j = torch.cat([torch.arange(k) for k in K]).cuda()
    return {"case": case, "pool": pool, "weights": weights.view(num_pages, page), "positions": positions.view(num_pages, page),
            "table": table, "seqlens": seqlens, "lens": lens, "next": torch.tensor(nxt, dtype=torch.int32, device="cuda"),
            "flat_b": flat_b, "flat_j": flat_j}


def prepare(case, seed):
    return {"moe_few": _prepare_moe, "accumulate": _prepare_accumulate, "evict": _prepare_evict}[case["op"]](case, seed)


# ------------------------------------------------------------------------------------------------- plain forms, in 32 bits
def _plain_moe(st):
    case, x = st["case"], st["x"].float()
    T, E, k = case["T"], case["E"], case["k"]
    logits = st["x"].double() @ st["Wg"].double()                      # two experts may lie within a rounding of each other
    p = torch.exp(logits - logits.max(dim=1, keepdim=True).values)
    top, idx = torch.sort(p, dim=1, descending=True, stable=True)      # ties: the lower expert first
    top, idx = top[:, :k], idx[:, :k]
    w = (top / top.sum(dim=1, keepdim=True)).float()

    def mlp(rows, W1, W3, W2):
        a = rows @ W1.float()
        return (a / (1.0 + torch.exp(-a)) * (rows @ W3.float())) @ W2.float()
    y = torch.zeros(T, case["d"], device=x.device)
    if T * k < E:                                                      # fewer choices than experts: one choice at a time
        for t in range(T):
            for j in range(k):
                e = idx[t, j:j + 1]
                W1, W3, W2 = (st[n].index_select(0, e)[0] for n in ("W1", "W3", "W2"))
                y[t] += w[t, j] * mlp(x[t:t + 1], W1, W3, W2)[0]
    else:
        gate = torch.zeros(T, E, device=x.device).scatter_(1, idx, w)
        for e in range(E):
            y += gate[:, e:e + 1] * mlp(x, st["W1"][e], st["W3"][e], st["W2"][e])
    if st["shared"] is not None:
        y += mlp(x, *st["shared"])
    return y.to(st["x"].dtype)


def _plain_accumulate(st):
    case = st["case"]
    H, Sq, d, page = case["H"], case["Sq"], case["d"], case["page"]
    out = st["weights"].clone().view(-1)
    flat = st["pool"].view(-1, d)
    for b, n in enumerate(st["lens"]):
        rows = _rows(st["table"][b], n, page)
        keys = flat[rows].float()
        q = st["Q"][b].reshape(H * Sq, d).float()
        m, l = st["m"][b].reshape(-1, 1), st["l"][b].reshape(-1, 1)
        got = torch.zeros(n, device=out.device)
        step = max(1, (1 << 27) // n)
        vis = None if Sq == 1 else _visible(n, Sq, H, out.device)
        for r in range(0, H * Sq, step):
            p = torch.exp(q[r:r + step] @ keys.T * st["scale"] - m[r:r + step]) / l[r:r + step]
            if vis is not None:
                p = torch.where(vis[r:r + step], p, torch.zeros_like(p))
            got += p.sum(dim=0)
        out[rows] += got
    return out.view_as(st["weights"])


def _plain_evict(st):
    case = st["case"]
    page, keep, lens = case["page"], case["keep"], st["lens"]
    table, dev = st["table"], st["pool"].device
    B, n_max = len(lens), max(lens)
    weights, positions = st["weights"].clone().view(-1), st["positions"].clone().view(-1)
    flat = st["pool"].view(-1, case["d"])
    t = torch.arange(n_max, device=dev)
    phys = table.long()[:, t // page] * page + t % page                # [B, n_max]; rows past a sequence's end: unused
    n = st["seqlens"].long()[:, None]
    K = torch.clamp(n, max=keep)
    # newest rows always stay, then by weight, then the lower row
    key = weights[phys].double()
    key = torch.where(positions[phys] >= st["next"][:, None] - case["recent"], torch.full_like(key, float("inf")), key)
    key = torch.where(t[None, :] < n, key, torch.full_like(key, float("-inf")))
    order = torch.sort(key, dim=1, descending=True, stable=True).indices
    kept = torch.zeros(B, n_max, dtype=torch.bool, device=dev)
    kept.scatter_(1, order, (t[None, :] < K))
    # survivors from behind row K take the places of evicted rows in front of it, both in ascending order
    hole = (t[None, :] < K) & ~kept
    mover = (t[None, :] >= K) & kept
    spare = torch.full((B, n_max + 1), -1, dtype=torch.long, device=dev)
    rank = torch.cumsum(mover, dim=1) - 1
    spare.scatter_(1, torch.where(mover, rank, torch.full_like(rank, n_max)), t.expand(B, n_max))
    hrank = torch.where(hole, torch.cumsum(hole, dim=1) - 1, torch.full_like(rank, n_max))
    src = torch.where(hole, spare.gather(1, hrank), t.expand(B, n_max))
    src = torch.where(t[None, :] < K, src, torch.full_like(src, -1))
    src = torch.cat((src, torch.full((B, max(0, keep - n_max)), -1, dtype=torch.long, device=dev)), dim=1)[:, :keep]
    fb, fj = st["flat_b"], st["flat_j"]
    to, frm = phys[fb, fj], phys[fb, src[fb, fj]]
    flat[to] = flat[frm]
    weights[to] = weights[frm]
    positions[to] = positions[frm]
    return {"pool": st["pool"], "weights": weights.view_as(st["weights"]), "positions": positions.view_as(st["positions"]),
            "kept": src.to(torch.int32), "seqlens": K[:, 0].to(torch.int32)}


# -------------------------------------------------------------------------------------------------- the library's operators
def _lib():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ds-flashdmla-moe_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import flashdmla
    return flashdmla


def _own(st):
    case = st["case"]
    F = _lib()
    if case["op"] == "moe_few":
        return F.moe_few(st["x"], st["Wg"], st["W1"], st["W3"], st["W2"], case["k"], st["shared"])
    if case["op"] == "accumulate":
        weights = st["weights"].clone()                                # the operator adds in place
        F.accumulate_weights(st["Q"], st["pool"], st["table"], st["seqlens"], st["m"], st["l"], weights, st["scale"])
        return weights
    weights, positions = st["weights"].clone(), st["positions"].clone()
    kept, seqlens = F.cache_evict(st["pool"], weights, positions, st["table"], st["seqlens"], st["next"], case["keep"],
                                  case["recent"])
    return {"pool": st["pool"], "weights": weights, "positions": positions, "kept": kept, "seqlens": seqlens}


def run(state):
    if own:
        return _own(state)
    return {"moe_few": _plain_moe, "accumulate": _plain_accumulate, "evict": _plain_evict}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------- the definition, in 64 bits
def _exact_moe(case, st):
    x = st["x"].double()
    z = x @ st["Wg"].double()
    prob = torch.softmax(z, dim=1)
    out = torch.zeros_like(x)
    chosen = [sorted(range(case["E"]), key=lambda e: (-row[e], e))[: case["k"]] for row in prob.tolist()]

    def ffn(rows, W1, W3, W2):
        a = rows @ W1.double()
        return ((a * torch.sigmoid(a)) * (rows @ W3.double())) @ W2.double()
    users = {}
    for t, es in enumerate(chosen):
        for e in es:
            users.setdefault(e, []).append(t)
    total = torch.stack([prob[t, es].sum() for t, es in enumerate(chosen)])
    for e, ts in sorted(users.items()):
        rows = torch.tensor(ts, device=x.device)
        share = prob[rows, e] / total[rows]
        out[rows] += share[:, None] * ffn(x[rows], st["W1"][e], st["W3"][e], st["W2"][e])
    if st["shared"] is not None:
        out += ffn(x, *st["shared"])
    return out


def _exact_accumulate(case, st):
    if work(case)["flops"] > 4e12:
        return None
    H, Sq, page = case["H"], case["Sq"], case["page"]
    out = st["weights"].double()
    for b, n in enumerate(st["lens"]):
        q = st["Q"][b].reshape(H, Sq, case["d"]).double()
        pages = st["table"][b].tolist()
        for lo in range(0, n, page):
            rows = min(page, n - lo)
            pg = pages[lo // page]
            s = torch.einsum("hqd,td->hqt", q, st["pool"][pg, :rows].double()) * st["scale"]
            p = torch.exp(s - st["m"][b].reshape(H, Sq, 1).double()) / st["l"][b].reshape(H, Sq, 1).double()
            key = torch.arange(lo, lo + rows, device=p.device)
            limit = torch.arange(Sq, device=p.device) + n - Sq
            p = p.masked_fill(key[None, None, :] > limit[None, :, None], 0.0)
            out[pg, :rows] += p.sum(dim=(0, 1))
    return out


def _exact_evict(case, st):
    page, keep, recent, d = case["page"], case["keep"], case["recent"], case["d"]
    weights, positions = st["weights"].double().view(-1).cpu().numpy(), st["positions"].view(-1).cpu().numpy()
    pool, table, nxt = st["pool"].double().view(-1, d), st["table"].cpu().numpy(), st["next"].tolist()
    kept = np.full((case["B"], keep), -1, dtype=np.int32)
    to, frm = [], []
    for b, n in enumerate(st["lens"]):
        row = np.arange(n)
        at = table[b][row // page].astype(np.int64) * page + row % page
        K = min(keep, n)
        # ascending by the last key first: protected rows, then the heavier ones, then the lower row
        best = np.lexsort((row, -weights[at], positions[at] < nxt[b] - recent))[:K]
        stays = np.zeros(n, dtype=bool)
        stays[best] = True
        holes, movers = np.flatnonzero(~stays[:K]), K + np.flatnonzero(stays[K:])
        kept[b, :K] = row[:K]
        kept[b, holes] = movers
        to.append(at[holes])
        frm.append(at[movers])
    to, frm = np.concatenate(to), np.concatenate(frm)
    weights[to], positions[to] = weights[frm].copy(), positions[frm].copy()
    pool[torch.from_numpy(to).cuda()] = pool[torch.from_numpy(frm).cuda()]
    dev = lambda a: torch.from_numpy(a).cuda()
    return {"pool": pool.view_as(st["pool"]), "weights": dev(weights).view_as(st["weights"]),
            "positions": dev(positions).view_as(st["positions"]), "kept": dev(kept),
            "seqlens": torch.tensor([min(keep, n) for n in st["lens"]], dtype=torch.int32, device="cuda")}


def exact(case, seed):
    st = prepare(case, seed)
    return {"moe_few": _exact_moe, "accumulate": _exact_accumulate, "evict": _exact_evict}[case["op"]](case, st)
