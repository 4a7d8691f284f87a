"""Operators of a bounded prefix cache: what they are measured on, in plain form and by
the framework's kernels.

  attend  attention of the new rows of one or several sequences over their paged caches
          (the rows' own keys are the last of the cache), with a sliding window and a few
          first tokens that stay visible, or over everything; the rows' log-sum-exp too
  mass    the attention weight every cached key got from those rows, added to what it had
  evict   the keys with the most weight kept, beside the first and the last ones, and
          moved together at the front of another cache (every layer and kv head)

Head counts are those of the workloads of ``specfold_amd.configs``, lengths their prefixes
(1024 to 16384), blocks of 32 tokens.  Every case is a dict of plain values with a
``kind``; where several sequences share a call, ``spread`` draws their lengths (up to
``prefix`` keys in front of up to ``rows`` new rows).  ``block`` 1 is a causal row, 32 the
block of a block-diffusion model (its rows see all of it); ``window`` 0 is no window.
"""

import math
import random

import torch

own = False

DEV = "cuda"
HD = 128
BF = torch.bfloat16

# heads, kv heads, layers of the named workloads
MODELS = {"1p5b": (12, 2, 28), "7b": (28, 4, 28), "8b": (32, 8, 32), "14b": (40, 8, 40)}


def listed():
    return [
        # one token of eight conversations, each over its own cache
        dict(name="attend_8b_token_x8", kind="attend", model="8b", seqs=8, rows=1, prefix=8192,
             block=1, window=0, sinks=0, page=16, spread=1),
        # one token of one long conversation that sees a window and the first tokens: latency
        dict(name="attend_14b_token_window", kind="attend", model="14b", seqs=1, rows=1,
             prefix=16384, block=1, window=1024, sinks=4, page=16, spread=0),
        # the default workload's block commit, four sequences at once
        dict(name="attend_7b_block_x4", kind="attend", model="7b", seqs=4, rows=32, prefix=2048,
             block=32, window=0, sinks=0, page=16, spread=2),
        # turns of four conversations of unlike lengths, ragged, causal
        dict(name="attend_8b_turns_x4", kind="attend", model="8b", seqs=4, rows=999, prefix=4096,
             block=1, window=0, sinks=0, page=16, spread=3),
        # a long prompt under a window
        dict(name="attend_14b_prompt_window", kind="attend", model="14b", seqs=1, rows=8192,
             prefix=0, block=32, window=2048, sinks=4, page=16, spread=0),
        # a long prompt that sees everything before it
        dict(name="attend_7b_prompt", kind="attend", model="7b", seqs=1, rows=8192, prefix=0,
             block=32, window=0, sinks=0, page=64, spread=0),
        # a decoded token's weights over a cache near its budget
        dict(name="mass_8b_token_x8", kind="mass", model="8b", seqs=8, rows=1, prefix=4096,
             block=1, window=0, sinks=0, page=16, spread=4),
        # a block's weights over a long cache
        dict(name="mass_14b_block", kind="mass", model="14b", seqs=1, rows=32, prefix=16384,
             block=32, window=0, sinks=0, page=16, spread=0),
        # a prompt's weights, which its first eviction goes by
        dict(name="mass_7b_prompt", kind="mass", model="7b", seqs=1, rows=4096, prefix=0,
             block=32, window=0, sinks=0, page=16, spread=0),
        # a small cache a little over its budget
        dict(name="evict_1p5b", kind="evict", model="1p5b", layers=28, length=1056, keep=1024,
             sinks=4, recent=256, page=16),
        # a prompt cut to a quarter, an odd length
        dict(name="evict_7b", kind="evict", model="7b", layers=28, length=4095, keep=1001,
             sinks=4, recent=512, page=16),
        # the long prefix cut to half
        dict(name="evict_14b", kind="evict", model="14b", layers=40, length=16384, keep=8192,
             sinks=4, recent=1024, page=64),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "mass", "evict"])
    model = rng.choice(list(MODELS))
    c = dict(kind=kind, model=model, page=rng.choice([16, 16, 32, 64, 128]))
    if kind == "evict":
        length = _log_int(rng, 64, 8192)
        keep = rng.randint(max(1, length // 8), length)
        sinks = min(rng.choice([0, 1, 4]), keep)
        c.update(layers=rng.randint(1, MODELS[model][2]), length=length, keep=keep, sinks=sinks,
                 recent=rng.randint(0, (keep - sinks) // 2))
        return c
    shape = rng.choice(["token", "block", "rows"])
    rows = {"token": 1, "block": rng.randint(2, 64), "rows": _log_int(rng, 33, 2048)}[shape]
    seqs = rng.randint(1, 8 if rows <= 512 else 2)
    c.update(seqs=seqs, rows=rows, block=rng.choice([1, 32]),
             prefix=_log_int(rng, 64, 16384 if rows <= 512 else 4096),
             spread=rng.randint(1, 10 ** 6))
    if rng.random() < 0.5:
        c.update(window=_log_int(rng, 32, 4096), sinks=rng.choice([0, 1, 4, 17]))
    else:
        c.update(window=0, sinks=0)
    return c


# ---- lengths and masks ----------------------------------------------------------------------


def _lengths(case):
    """(new rows, cached keys with them) of every sequence; the first has the most."""
    rng = random.Random(case["spread"])
    out = []
    for i in range(case["seqs"]):
        f, g = (1.0, 1.0) if i == 0 else (rng.random(), rng.random())
        n = 1 + int(f * (case["rows"] - 1))
        out.append((n, n + int(g * case["prefix"])))
    return out


def _limits(case, n, P, device="cpu"):
    """Of every row: the end of the keys it sees, and the first it sees behind the sinks."""
    m = torch.arange(n, device=device)
    p = P - n + m
    end = P - n + ((m // case["block"] + 1) * case["block"]).clamp(max=n)
    lo = (p - case["window"] + 1).clamp(min=0) if case["window"] else torch.zeros_like(p)
    return end, lo


# ---- inputs ---------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _rnd(g, *shape, std=1.0):
    return torch.empty(*shape, dtype=BF, device=DEV).normal_(0.0, std, generator=g)


def _ws(n):
    return torch.empty(max(int(n), 256), dtype=torch.uint8, device=DEV)


def _cached(case, seed):
    """The sequences' pages ([pages, Hkv, page, hd] K and V), page tables and queries."""
    H, Hkv, _ = MODELS[case["model"]]
    g = _gen(seed)
    cpu = torch.Generator().manual_seed(int(seed))
    u = _rnd(g, Hkv, HD)       # what queries share, and the first keys answer to
    seqs, qs = [], []
    for n, P in _lengths(case):
        npg = -(-P // case["page"])
        k, v = (_rnd(g, npg, Hkv, case["page"], HD) for _ in range(2))
        table = torch.randperm(npg, generator=cpu).to(torch.int32)
        k[int(table[0]), :, :min(4, P)] += 0.5 * u[:, None]
        q = 1.5 * _rnd(g, n, Hkv, H // Hkv, HD).float() + 0.5 * u.float()[:, None]
        qs.append(q.to(BF).view(n, H * HD))
        seqs.append(dict(k=k, v=v, table=table.to(DEV), n=n, P=P))
    return seqs, torch.cat(qs)


def _rows_of(pages, table, P, h):
    """Keys (or values) 0 .. P - 1 of kv head h in order, [P, hd]."""
    return pages[table.long()][:, h].reshape(-1, HD)[:P]


def _scores(case, q, k, n, P, dtype):
    """[G, n, P] scores of q [n, G, hd] with what a row does not see at -inf."""
    s = torch.matmul(q.transpose(0, 1).to(dtype), k.to(dtype).t()) * HD ** -0.5
    end, lo = _limits(case, n, P, q.device)
    t = torch.arange(P, device=q.device)
    seen = (t < end[:, None]) & ((t < case["sinks"]) | (t >= lo[:, None]))
    return s.masked_fill_(~seen, -math.inf)


def _lse(case, seqs, q, dtype=torch.float32):
    """Log-sum-exp of every row's scores, [rows, H]."""
    H, Hkv, _ = MODELS[case["model"]]
    out, r = torch.empty(q.shape[0], H, dtype=dtype, device=DEV), 0
    for s in seqs:
        qs = q[r:r + s["n"]].view(s["n"], Hkv, H // Hkv, HD)
        for h in range(Hkv):
            x = _scores(case, qs[:, h], _rows_of(s["k"], s["table"], s["P"], h), s["n"], s["P"],
                        dtype)
            top = x.amax(-1)
            out[r:r + s["n"], h * (H // Hkv):(h + 1) * (H // Hkv)] = \
                (top + (x - top[..., None]).exp_().sum(-1).log()).t()
        r += s["n"]
    return out


def _masses(case, seqs, seed):
    """What every key had before, of each sequence [Hkv, P]."""
    g = _gen(seed + 31)
    Hkv = MODELS[case["model"]][1]
    return [torch.empty(Hkv, s["P"], device=DEV).exponential_(2.0, generator=g) for s in seqs]


def _evict_inputs(case, seed):
    _, Hkv, _ = MODELS[case["model"]]
    g = _gen(seed)
    cpu = torch.Generator().manual_seed(int(seed))
    L, P = case["layers"], case["length"]
    npg, nkeep = -(-P // case["page"]), -(-case["keep"] // case["page"])
    k, v = (_rnd(g, L, npg, Hkv, case["page"], HD) for _ in range(2))
    # a few keys carry most of the weight; keys that no row saw have none
    mass = torch.empty(L, Hkv, P, device=DEV).normal_(0.0, 2.0, generator=g).exp_()
    mass[torch.rand(L, Hkv, P, generator=g, device=DEV) < 0.25] = 0.0
    return dict(k=k, v=v, mass=mass, table=torch.randperm(npg, generator=cpu).to(torch.int32).to(DEV),
                table2=torch.randperm(nkeep, generator=cpu).to(torch.int32).to(DEV))


def _cache(layers, Hkv, page, k, v, table, length):
    """A framework cache that holds these pages."""
    from specfold_amd.kv_cache import PagedKVCache
    c = PagedKVCache(layers, Hkv, HD, table.numel() * page, page_size=page, device=DEV)
    c.k_pages.copy_(k)
    c.v_pages.copy_(v)
    c.page_table.copy_(table)
    c.advance(length)
    return c


def prepare(case, seed):
    H, Hkv, _ = MODELS[case["model"]]
    if case["kind"] == "evict":
        t = _evict_inputs(case, seed)
        L, keep, page = case["layers"], case["keep"], case["page"]
        s = dict(case=dict(case), **t)
        shape = (L, t["table2"].numel(), Hkv, page, HD)
        s["k2"], s["v2"] = (torch.zeros(shape, dtype=BF, device=DEV) for _ in range(2))
        if own:
            s["cache"] = _cache(L, Hkv, page, s.pop("k"), s.pop("v"), t["table"], case["length"])
            s["into"] = _cache(L, Hkv, page, s.pop("k2"), s.pop("v2"), t["table2"], 0)
            s["kept"] = torch.empty(L, Hkv, keep, dtype=torch.int32, device=DEV)
            s["mass2"] = torch.empty(L, Hkv, keep, device=DEV)
        return s
    seqs, q = _cached(case, seed)
    s = dict(case=dict(case), q=q)
    if case["kind"] == "mass":
        s["lse"], s["mass"] = _lse(case, seqs, q), _masses(case, seqs, seed)
        s["out"] = [torch.empty_like(m) for m in s["mass"]]
    else:
        s["o"] = torch.empty_like(q)
        s["lse"] = torch.empty(q.shape[0], H, device=DEV)
    if own:
        from specfold_amd import _lib
        from specfold_amd.kv_cache import PagedBatch
        s["batch"] = PagedBatch([_cache(1, Hkv, case["page"], x["k"], x["v"], x["table"], x["P"])
                                 for x in seqs], [x["n"] for x in seqs])
        s["ws"] = _ws(_lib.attn_window_workspace_bytes(q.shape[0], H) if case["kind"] == "attend"
                      else _lib.attn_key_mass_workspace_bytes(sum(x["P"] for x in seqs), Hkv))
    else:
        s["seqs"] = seqs
    return s


# ---- one pass -------------------------------------------------------------------------------


def run(s):
    case = s["case"]
    if own:
        return _run_own(s)
    if case["kind"] == "evict":
        return _evict_plain(s)
    H, Hkv, _ = MODELS[case["model"]]
    G, r = H // Hkv, 0
    for i, x in enumerate(s["seqs"]):
        n, P = x["n"], x["P"]
        qs = s["q"][r:r + n].view(n, Hkv, G, HD)
        for h in range(Hkv):
            sc = _scores(case, qs[:, h], _rows_of(x["k"], x["table"], P, h), n, P, torch.float32)
            heads = slice(h * G, (h + 1) * G)
            if case["kind"] == "attend":
                top = sc.amax(-1, keepdim=True)
                p = sc.sub_(top).exp_()
                z = p.sum(-1, keepdim=True)
                v = _rows_of(x["v"], x["table"], P, h).float()
                o = torch.matmul(p, v) / z
                s["o"][r:r + n].view(n, H, HD)[:, heads] = o.transpose(0, 1).to(BF)
                s["lse"][r:r + n, heads] = (top + z.log())[..., 0].t()
            else:
                p = sc.sub_(s["lse"][r:r + n, heads].t()[..., None]).exp_()
                s["out"][i][h] = s["mass"][i][h] + p.sum((0, 1))
        r += n
    return {"o": s["o"], "lse": s["lse"]} if case["kind"] == "attend" else list(s["out"])


def _run_own(s):
    from specfold_amd import _lib
    case = s["case"]
    H = MODELS[case["model"]][0]
    if case["kind"] == "evict":
        s["cache"].evict(s["mass"], case["keep"], sinks=case["sinks"], recent=case["recent"],
                         into=s["into"], kept=s["kept"], mass_out=s["mass2"])
        return {"k": s["into"].k_pages, "v": s["into"].v_pages, "kept": s["kept"],
                "mass": s["mass2"]}
    mask = dict(block=case["block"], window=case["window"], sinks=case["sinks"])
    if case["kind"] == "attend":
        _lib.attn_window(s["q"], s["batch"], 0, H, HD ** -0.5, s["o"], s["ws"], lse=s["lse"], **mask)
        return {"o": s["o"], "lse": s["lse"]}
    _lib.attn_key_mass(s["q"], s["lse"], s["batch"], 0, H, HD ** -0.5, s["out"], s["ws"],
                       mass_in=s["mass"], **mask)
    return list(s["out"])


def _kept(case, mass):
    """Ascending indices of the keys to keep, [L, Hkv, keep]: equal weights, the lower
    index first."""
    P, keep, sinks, recent = case["length"], case["keep"], case["sinks"], case["recent"]
    sinks, recent = min(sinks, P), min(recent, P)
    m = mass.clone()
    m[..., :sinks] = math.inf
    m[..., P - recent:] = math.inf
    return torch.sort(m, dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values


def _evict_plain(s):
    case = s["case"]
    L, Hkv, keep = s["mass"].shape[0], s["mass"].shape[1], case["keep"]
    page = case["page"]
    kept = _kept(case, s["mass"])
    li = torch.arange(L, device=DEV)[:, None, None]
    hi = torch.arange(Hkv, device=DEV)[None, :, None]
    at = torch.arange(keep, device=DEV)
    for src, dst in ((s["k"], s["k2"]), (s["v"], s["v2"])):
        dst[li, s["table2"].long()[at // page], hi, at % page] = \
            src[li, s["table"].long()[kept // page], hi, kept % page]
    return {"k": s["k2"], "v": s["v2"], "kept": kept.to(torch.int32),
            "mass": torch.gather(s["mass"], -1, kept)}


# ---- what a pass cannot do without ----------------------------------------------------------


def work(case):
    H, Hkv, _ = MODELS[case["model"]]
    if case["kind"] == "evict":
        n = case["layers"] * Hkv
        return {"bytes": n * (4 * case["length"] + case["keep"] * (2 * 2 * 2 * HD + 8)),
                "flops": n * case["length"]}
    pairs, keys, rows, held = 0, 0, 0, 0
    for n, P in _lengths(case):
        end, lo = _limits(case, n, P)
        first = torch.minimum(torch.full_like(lo, case["sinks"]), lo)
        pairs += int((end - lo + first).sum())
        keys += P - int(lo[0]) + min(case["sinks"], int(lo[0]))
        rows, held = rows + n, held + P
    if case["kind"] == "attend":
        return {"bytes": 4 * Hkv * HD * keys + rows * H * (4 * HD + 4), "flops": 4 * H * HD * pairs}
    return {"bytes": 2 * Hkv * HD * keys + rows * H * (2 * HD + 4) + 8 * Hkv * held,
            "flops": 2 * H * HD * pairs}


# ---- the same in 64 bits --------------------------------------------------------------------


def exact(case, seed):
    H, Hkv, _ = MODELS[case["model"]]
    G = H // Hkv
    if case["kind"] == "evict":
        t = _evict_inputs(case, seed)
        P, keep, page = case["length"], case["keep"], case["page"]
        first, last = min(case["sinks"], P), P - min(case["recent"], P)
        order = torch.argsort(-t["mass"][..., first:last].double(), dim=-1, stable=True) + first
        middle = order[..., :max(0, keep - first - (P - last))]
        L = case["layers"]
        ends = torch.cat([torch.arange(first, device=DEV), torch.arange(last, P, device=DEV)])
        kept = torch.cat([middle, ends.expand(L, Hkv, -1)], -1).sort(-1).values
        out = {"kept": kept.to(torch.int32), "mass": torch.gather(t["mass"].double(), -1, kept)}
        for name in ("k", "v"):
            y = torch.zeros(L, t["table2"].numel(), Hkv, page, HD, dtype=torch.float64, device=DEV)
            for l in range(L):
                for h in range(Hkv):
                    rows = t[name][l, :, h][t["table"].long()].reshape(-1, HD)[kept[l, h]].double()
                    full = rows.new_zeros(y.shape[1] * page, HD)
                    full[:keep] = rows
                    y[l, t["table2"].long(), h] = full.view(-1, page, HD)
            out[name] = y
        return {k: out[k] for k in ("k", "v", "kept", "mass")}
    seqs, q = _cached(case, seed)
    mass = case["kind"] == "mass"
    lse_in = _lse(case, seqs, q) if mass else None
    had = _masses(case, seqs, seed) if mass else None
    o = torch.empty(q.shape[0], H, HD, dtype=torch.float64, device=DEV)
    lse = torch.empty(q.shape[0], H, dtype=torch.float64, device=DEV)
    got, r = [], 0
    for i, x in enumerate(seqs):
        n, P = x["n"], x["P"]
        pos = torch.arange(P - n, P, device=DEV)
        t = torch.arange(P, device=DEV)
        blk = (pos - (P - n)) // case["block"]
        see = (t[None] < P - n) | ((t[None] - (P - n)) // case["block"] <= blk[:, None])
        if case["window"]:
            see &= (pos[:, None] - t[None] < case["window"]) | (t[None] < case["sinks"])
        if mass:
            got.append(had[i].double())
        for hq in range(H):
            h = hq // G
            k = x["k"][x["table"].long()][:, h].reshape(-1, HD)[:P].double()
            sc = q[r:r + n].view(n, H, HD)[:, hq].double() @ k.t() / math.sqrt(HD)
            sc.masked_fill_(~see, -math.inf)
            if mass:
                got[i][h] += (sc - lse_in[r:r + n, hq].double()[:, None]).exp().sum(0)
            else:
                v = x["v"][x["table"].long()][:, h].reshape(-1, HD)[:P].double()
                lse[r:r + n, hq] = torch.logsumexp(sc, -1)
                o[r:r + n, hq] = torch.softmax(sc, -1) @ v
        r += n
    return got if mass else {"o": o.view(q.shape[0], H * HD), "lse": lse}
