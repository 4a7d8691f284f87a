"""Plain 64-bit forms of sf_attn_window, sf_attn_key_mass and sf_kv_evict, the bounds their
results are held to, and the calls over paged caches; on any device (the simulator's tests
run them on the CPU)."""

import math

import torch

from specfold_amd.kv_cache import PagedBatch, PagedKVCache

HD = 128
BF = torch.bfloat16


def seen(n, P, block, window, sinks, device="cpu"):
    """[n, P] of truth values: which keys each row sees."""
    t = torch.arange(P, device=device)
    m = torch.arange(n, device=device)[:, None]
    p = P - n + m
    end = P - n + torch.clamp((m // block + 1) * block, max=n)
    ok = t < end
    if window:
        ok = ok & ((t < sinks) | (t > p - window))
    return ok


def plain_attention(q, k, v, block=1, window=0, sinks=0, scaling=HD ** -0.5):
    """q [n, H, hd], k, v [Hkv, P, hd] -> o, lse, and of every output the bound of its error:
    weights and output rounded to bf16 (2^-8 each), fp32 scores and sums."""
    n, H, _ = q.shape
    Hkv, P, _ = k.shape
    ok = seen(n, P, block, window, sinks, q.device)
    o, tol = (torch.empty(n, H, HD, dtype=torch.float64, device=q.device) for _ in range(2))
    lse, tol_l = (torch.empty(n, H, dtype=torch.float64, device=q.device) for _ in range(2))
    for h in range(H):
        kk, vv = k[h * Hkv // H].double(), v[h * Hkv // H].double()
        s = (q[:, h].double() @ kk.t() * scaling).masked_fill(~ok, -math.inf)
        w = torch.softmax(s, -1)
        o[:, h] = w @ vv
        lse[:, h] = torch.logsumexp(s, -1)
        # a score: 128 products summed in fp32 (2^-24 a step, of at most the sum of their
        # magnitudes), scaled, and the exponent's two roundings
        mag = (q[:, h].double().abs() @ kk.abs().t() * scaling).masked_fill(~ok, 0).amax(-1)
        eps = 136 * 2.0 ** -24 * mag + 2.0 ** -21
        sums = P * 2.0 ** -24
        wv = w @ vv.abs()
        tol[:, h] = 2 ** -8 * o[:, h].abs() + (2 ** -8 + 2 * eps + 2 * sums)[:, None] * wv * 1.01
        tol_l[:, h] = eps + sums + 2.0 ** -23 * (lse[:, h].abs() + s.amax(-1).abs()) + 2.0 ** -22
    return o, lse, tol, tol_l


def plain_mass(q, lse, k, block=1, window=0, sinks=0, scaling=HD ** -0.5):
    """[Hkv, P] sums of the weights and their bounds."""
    n, H, _ = q.shape
    Hkv, P, _ = k.shape
    ok = seen(n, P, block, window, sinks, q.device)
    out, tol = (torch.zeros(Hkv, P, dtype=torch.float64, device=q.device) for _ in range(2))
    for h in range(H):
        kk = k[h * Hkv // H].double()
        s = q[:, h].double() @ kk.t() * scaling
        w = torch.exp((s - lse[:, h].double()[:, None]).masked_fill(~ok, -math.inf))
        mag = (q[:, h].double().abs() @ kk.abs().t() * scaling).amax()
        eps = 136 * 2.0 ** -24 * mag + 2.0 ** -22 * lse[:, h].abs().max().double() + 2.0 ** -21
        out[h * Hkv // H] += w.sum(0)
        tol[h * Hkv // H] += w.sum(0) * (eps + n * H * 2.0 ** -24)
    return out, tol


def plain_kept(mass, length, keep, sinks, recent):
    """[L, Hkv, keep] ascending slots: first, last, then the largest mass, ties the lower;
    one (layer, head) after the other, in Python."""
    L, Hkv, _ = mass.shape
    out = torch.empty(L, Hkv, keep, dtype=torch.int64)
    for l in range(L):
        for h in range(Hkv):
            m = mass[l, h, :length].tolist()
            ends = list(range(sinks)) + list(range(length - recent, length))
            mid = sorted(range(sinks, length - recent),
                         key=lambda t: (0 if m[t] != m[t] else 1, -m[t] if m[t] == m[t] else 0, t))
            out[l, h] = torch.tensor(sorted(ends + mid[:keep - sinks - recent]))
    return out


def make_seqs(shapes, H, Hkv, seed, device, page=16, order="shuffled", std=1.0, spare=40):
    """Sequences [(n, P), ...]: queries [rows, H, hd], per-sequence k, v [Hkv, P, hd] and
    caches of one layer that hold them (with room of NaN behind the length)."""
    g = torch.Generator().manual_seed(seed)
    caches, ks, vs = [], [], []
    for i, (n, P) in enumerate(shapes):
        k, v = (torch.randn(Hkv, P, HD, generator=g).to(BF).to(device) for _ in range(2))
        c = PagedKVCache(1, Hkv, HD, P + spare, page_size=page, device=device, page_order=order,
                         seed=seed + i)
        c.k_pages.fill_(math.nan)
        c.v_pages.fill_(math.nan)
        idx = c.page_table.long()
        for src, dst in ((k, c.k_pages), (v, c.v_pages)):
            full = torch.full((Hkv, c.capacity, HD), math.nan, dtype=BF, device=device)
            full[:, :P] = src
            dst[0][idx] = full.view(Hkv, -1, page, HD).transpose(0, 1)
        c.advance(P)
        caches.append(c)
        ks.append(k)
        vs.append(v)
    rows = sum(n for n, _ in shapes)
    q = (std * torch.randn(max(rows, 1), H, HD, generator=g)).to(BF).to(device)
    return q, ks, vs, caches


def run_window(lib, q, caches, ns, H, block=1, window=0, sinks=0, scaling=HD ** -0.5, lse=True,
               guard=2, stream=None, li=0):
    """o [rows, H, hd], lse [rows, H]; rows behind the batch's must stay as they were."""
    rows = sum(ns)
    dev = q.device
    o = torch.full((rows + guard, H * HD), 7.0, dtype=BF, device=dev)
    ls = torch.full((rows + guard, H), 7.0, device=dev) if lse else None
    ws = torch.full((lib.attn_window_workspace_bytes(rows, H),), 255, dtype=torch.uint8, device=dev)
    batch = PagedBatch(caches, ns)
    for _ in range(2):      # twice through one workspace
        lib.attn_window(q, batch, li, H, scaling, o, ws, lse=ls, block=block, window=window,
                        sinks=sinks, stream=stream)
    assert torch.all(o[rows:] == 7.0)
    if lse:
        assert torch.all(ls[rows:] == 7.0)
        ls = ls[:rows]
    return o[:rows].view(rows, H, HD), ls


def check_window(lib, shapes, H, Hkv, block, window, sinks, device, seed=0, page=16, std=1.0,
                 order="shuffled"):
    q, ks, vs, caches = make_seqs(shapes, H, Hkv, seed, device, page=page, std=std, order=order)
    ns = [n for n, _ in shapes]
    o, lse = run_window(lib, q, caches, ns, H, block, window, sinks)
    r = 0
    for (n, P), k, v in zip(shapes, ks, vs):
        if n:
            ro, rl, tol, tol_l = plain_attention(q[r:r + n], k, v, block, window, sinks)
            d = (o[r:r + n].double() - ro).abs()
            assert torch.all(d <= tol), (n, P, float((d / tol).max()))
            dl = (lse[r:r + n].double() - rl).abs()
            assert torch.all(dl <= tol_l), (n, P, float((dl / tol_l).max()))
        r += n


def check_mass(lib, shapes, H, Hkv, block, window, sinks, device, seed=0, page=16, decay=1.0,
               inplace=False, fresh=False):
    q, ks, vs, caches = make_seqs(shapes, H, Hkv, seed, device, page=page)
    ns = [n for n, _ in shapes]
    rows = sum(ns)
    g = torch.Generator().manual_seed(seed + 5)
    lse = torch.full((max(rows, 1), H), 7.0, device=device)
    r = 0
    for (n, P), k, v in zip(shapes, ks, vs):
        if n:
            lse[r:r + n] = plain_attention(q[r:r + n], k, v, block, window, sinks)[1].float()
        r += n
    had = [torch.rand(Hkv, P + 9, generator=g).to(device) for _, P in shapes]
    was = [h.clone() for h in had]
    out = had if inplace else [torch.full((Hkv, P + 3), 7.0, device=device) for _, P in shapes]
    ws = torch.full((lib.attn_key_mass_workspace_bytes(sum(P for _, P in shapes), Hkv),), 255,
                    dtype=torch.uint8, device=device)
    batch = PagedBatch(caches, ns)
    lib.attn_key_mass(q, lse, batch, 0, H, HD ** -0.5, out, ws, mass_in=None if fresh else had,
                      decay=decay, block=block, window=window, sinks=sinks)
    r = 0
    for i, ((n, P), k) in enumerate(zip(shapes, ks)):
        ref, tol = plain_mass(q[r:r + n], lse[r:r + n], k, block, window, sinks) if n else \
            (torch.zeros(Hkv, P, dtype=torch.float64, device=device),) * 2
        base = torch.zeros_like(ref) if fresh else float(torch.tensor(decay)) * was[i][:, :P].double()
        ref = ref + base
        d = (out[i][:, :P].double() - ref).abs()
        bound = tol + 2.0 ** -23 * (ref.abs() + base) + 1e-30
        assert torch.all(d <= bound), (n, P, float((d / bound).max()))
        assert torch.equal(out[i][:, P:], was[i][:, P:]) if inplace else torch.all(out[i][:, P:] == 7.0)
        r += n


def check_evict(L, Hkv, length, keep, sinks, recent, device, into, page=16, page2=None, seed=0,
                mass=None):
    g = torch.Generator().manual_seed(seed)
    c = PagedKVCache(L, Hkv, HD, length + 30, page_size=page, device=device, page_order="shuffled",
                     seed=seed)
    bits = torch.randint(-2 ** 15, 2 ** 15, c.k_pages.shape, generator=g, dtype=torch.int16)
    c.k_pages.copy_(bits.view(BF).to(device))
    c.v_pages.copy_(bits.flip(0, 1, 2, 3, 4).view(BF).to(device))
    c.advance(length)
    if mass is None:
        mass = torch.randn(L, Hkv, length + 11, generator=g).exp()
        mass = torch.where(torch.rand(mass.shape, generator=g) < 0.3, 0.5, mass)   # ties
    was = mass.clone()
    mass = mass.to(device)
    # the cache whole, in logical order, as 16-bit patterns
    def whole(x):
        full = [pages[:, x.page_table.long()].transpose(2, 3).reshape(L, x.capacity, Hkv, HD)
                .cpu().view(torch.int16) for pages in (x.k_pages, x.v_pages)]
        return full
    before = whole(c)
    kw, to = {}, c
    if into:
        to = PagedKVCache(L, Hkv, HD, keep + 20, page_size=page2 or page, device=device,
                          page_order="shuffled", seed=seed + 1)
        out = torch.full((L, Hkv, keep + 5), 7.0, device=device)
        kw = dict(into=to, mass_out=out)
    kept = c.evict(mass, keep, sinks=sinks, recent=recent, **kw).cpu().long()
    ref = plain_kept(was, length, keep, sinks, recent)
    assert torch.equal(kept, ref)
    after = whole(to)
    at = ref.transpose(1, 2)[..., None].expand(L, keep, Hkv, HD)
    for b, a in zip(before, after):
        assert torch.equal(a[:, :keep], torch.gather(b, 1, at))
        if into:
            assert torch.all(a[:, keep:] == 0)
        else:
            assert torch.equal(a[:, keep:], b[:, keep:])
    km = torch.gather(was, 2, ref)
    got = (out if into else mass).cpu()
    assert torch.equal(got[..., :keep].view(torch.int32), km.view(torch.int32))
    if into:
        assert torch.all(got[..., keep:] == 7.0)
        assert torch.equal(mass.cpu().view(torch.int32), was.view(torch.int32))
        for b, a in zip(before, whole(c)):
            assert torch.equal(a, b)
    else:
        assert torch.all(got[..., keep:length] == 0)
        assert torch.equal(got[..., length:], was[..., length:])
    assert to.length == keep and to.position == length
    assert int(to.length_dev) == keep and int(to.position_dev) == length
