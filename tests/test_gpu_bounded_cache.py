"""sf_attn_window, sf_attn_key_mass and sf_kv_evict on the GPU against 64-bit forms, alone,
captured, on other streams, and together through the engine."""

import math

import pytest
import torch

from specfold_amd import _lib
from specfold_amd.engine import FoldedVerifyEngine
from specfold_amd.kv_cache import PagedBatch, PagedKVCache
from tests.bounded_cache import (BF, HD, check_evict, check_mass, check_window, make_seqs,
                                 plain_attention, plain_mass, run_window, seen)
from tests.helpers import SHAPE_G2, SHAPE_N8, build_nld, build_qwen2, to_gpu_model

pytestmark = pytest.mark.gpu

# (n, P) of each sequence, H, Hkv, block, window, sinks, page
WINDOW = [
    ([(1, 1)], 28, 4, 1, 0, 0, 16),
    ([(1, 8001)], 32, 8, 1, 0, 0, 16),
    ([(1, 16384)], 40, 8, 1, 1024, 4, 16),
    ([(1, 32768)], 12, 2, 1, 0, 0, 128),
    ([(1, p) for p in (4096, 17, 1, 900, 2222, 64, 65, 4095)], 32, 8, 1, 0, 0, 16),
    ([(1, 37 * i + 1) for i in range(32)], 8, 2, 1, 300, 5, 32),
    ([(2, 5000), (3, 70), (0, 0), (4, 4)], 28, 4, 1, 0, 0, 16),
    ([(7, 3000)], 16, 1, 1, 0, 0, 16),
    ([(32, 2080)] * 4, 28, 4, 32, 0, 0, 16),
    ([(32, 16416)], 40, 8, 32, 0, 0, 16),
    ([(32, 2080), (5, 700), (64, 64), (1, 900)], 12, 2, 32, 512, 4, 64),
    ([(999, 5000), (70, 170), (500, 500)], 32, 8, 1, 0, 0, 16),
    ([(1000, 1000)], 28, 4, 32, 0, 0, 16),
    ([(1025, 2049)], 40, 8, 32, 333, 17, 16),
    ([(2000, 2000)], 12, 2, 1, 64, 4, 32),
    ([(700, 1500)], 7, 7, 1, 1, 0, 16),
    ([(600, 1800)], 16, 1, 16, 200, 130, 16),
    ([(2047, 2111)], 28, 4, 64, 1000, 1, 128),
    # (few queries over 9 to 36 stages of keys, and just outside)
    ([(1, p) for p in (1151, 289, 288, 257, 256, 33, 1, 1152)], 32, 8, 1, 0, 0, 16),
    ([(1, 1152), (1, 1153)], 40, 8, 1, 0, 0, 16),
    ([(2, 1030), (3, 900)], 40, 8, 1, 500, 70, 32),
    ([(2, 900)], 16, 1, 2, 0, 0, 128),
]


@pytest.mark.parametrize("shapes,H,Hkv,block,window,sinks,page", WINDOW)
def test_window(shapes, H, Hkv, block, window, sinks, page):
    check_window(_lib, shapes, H, Hkv, block, window, sinks, "cuda", seed=len(shapes) + window,
                 page=page)


@pytest.mark.parametrize("shapes,H,Hkv,block", [([(300, 900)], 28, 4, 32), ([(1, 3000)], 32, 8, 1),
                                                ([(32, 6000)], 40, 8, 32)])
def test_window_large_scores(shapes, H, Hkv, block):
    """Scores far apart: the running maximum moves from chunk to chunk."""
    check_window(_lib, shapes, H, Hkv, block, 0, 0, "cuda", std=6.0)


@pytest.mark.parametrize("n,P,block,window,sinks,at", [
    (64, 64, 32, 0, 0, 40), (1000, 1077, 1, 0, 0, 600), (1024, 2048, 32, 256, 4, 1500),
    (200, 5200, 16, 0, 0, 5199), (129, 129, 64, 0, 0, 128), (700, 900, 1, 100, 40, 330),
    (2, 3000, 1, 0, 0, 2999), (32, 4000, 32, 100, 4, 3880), (2, 500, 1, 0, 0, 499),
    (2, 900, 1, 300, 4, 599)])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_hidden_key_not_finite(n, P, block, window, sinks, at, bad):
    """A value or key that is not finite reaches the rows that see it (a value: in its
    dims), and no other."""
    H, Hkv = 28, 4
    q, ks, vs, _ = make_seqs([(n, P)], H, Hkv, n + P, "cuda")
    k, v, kz, vz = ks[0].clone(), vs[0].clone(), ks[0].clone(), vs[0].clone()
    v[1, at, [3, 64]], vz[1, at, [3, 64]] = bad, 0
    if bad != bad:
        k[1, at, 5], kz[1, at, 5] = bad, 0
    c = PagedKVCache(1, Hkv, HD, P, device="cuda", page_order="shuffled", seed=2)
    c.load_dense([(k[None], v[None])])
    o, lse = run_window(_lib, q, [c], [n], H, block, window, sinks)
    ro, rl, tol, tol_l = plain_attention(q[:n], kz, vz, block, window, sinks)
    see = seen(n, P, block, window, sinks, "cuda")[:, at]
    heads = torch.arange(H, device="cuda") // (H // Hkv) == 1
    ok = (o.double() - ro).abs() <= tol
    assert torch.all(ok[~see]) and torch.all(ok[:, ~heads])
    assert not torch.any(o[see][:, heads][..., [3, 64]].isfinite())
    if bad == bad:
        ok[..., [3, 64]] = True
        assert torch.all(ok)
        assert torch.all((lse.double() - rl).abs() <= tol_l)


def test_window_repeats():
    """The same call gives the same bits."""
    q, ks, vs, caches = make_seqs([(300, 1000), (1, 4000), (32, 3000)], 28, 4, 5, "cuda")
    ns = [300, 1, 32]
    ref = run_window(_lib, q, caches, ns, 28, 32, 700, 4)
    for _ in range(3):
        got = run_window(_lib, q, caches, ns, 28, 32, 700, 4)
        assert torch.equal(ref[0], got[0]) and torch.equal(ref[1], got[1])


def test_sequences_do_not_meet():
    """A sequence's rows are the same alone and beside others."""
    shapes = [(32, 2000), (1, 3000), (200, 400)]
    q, ks, vs, caches = make_seqs(shapes, 32, 8, 6, "cuda")
    o, lse = run_window(_lib, q, caches, [n for n, _ in shapes], 32, 32, 0, 0)
    r = 0
    for (n, P), k, v in zip(shapes, ks, vs):
        ro, rl, tol, tol_l = plain_attention(q[r:r + n], k, v, 32)
        assert torch.all((o[r:r + n].double() - ro).abs() <= tol)
        r += n


MASS = [
    ([(1, 1)], 28, 4, 1, 0, 0, 16),
    ([(1, 8001)], 32, 8, 1, 0, 0, 16),
    ([(1, p) for p in (4096, 17, 1, 900, 64, 65)] + [(0, 300), (0, 0)], 32, 8, 1, 0, 0, 16),
    ([(1, 16384)], 40, 8, 1, 1024, 4, 16),
    ([(32, 2080), (5, 700), (64, 64)], 12, 2, 32, 512, 4, 64),
    ([(32, 16416)], 40, 8, 32, 0, 0, 16),
    ([(999, 3000), (70, 170)], 28, 4, 1, 0, 0, 16),
    ([(1025, 2049)], 40, 8, 32, 333, 17, 128),
    ([(600, 1800)], 16, 1, 16, 200, 130, 16),
    # (ranges of more stages than are summed lane by lane)
    ([(2500, 2600)], 28, 4, 32, 0, 0, 16),
]


@pytest.mark.parametrize("shapes,H,Hkv,block,window,sinks,page", MASS)
@pytest.mark.parametrize("how", ["fresh", "add", "inplace"])
def test_mass(shapes, H, Hkv, block, window, sinks, page, how):
    check_mass(_lib, shapes, H, Hkv, block, window, sinks, "cuda", page=page,
               decay=0.75 if how == "inplace" else 1.0, inplace=how == "inplace",
               fresh=how == "fresh")


EVICT = [
    (1, 1, 1, 1, 0, 0), (3, 4, 4096, 1024, 4, 256), (2, 8, 4095, 1001, 4, 500),
    (2, 2, 4097, 4096, 0, 1), (1, 8, 16384, 8192, 4, 1024), (1, 2, 32768, 20000, 0, 0),
    (1, 2, 32767, 1, 0, 0), (4, 2, 777, 776, 100, 100), (2, 4, 600, 300, 150, 150),
    (1, 1, 1025, 513, 1, 0),
]


@pytest.mark.parametrize("case", EVICT)
@pytest.mark.parametrize("into", [False, True])
def test_evict(case, into):
    check_evict(*case, "cuda", into, page2=64 if case[2] % 2 else None)


def _work_between():
    """Eager work between replays."""
    return float((torch.ones(1 << 16, device="cuda") * 3).sum())


def test_captured_and_replayed():
    """Attention, mass and eviction captured into one graph: every replay, with new inputs in
    the same buffers, gives what the eager calls give."""
    H, Hkv, P, keep = 28, 4, 1500, 700
    shapes = [(64, P), (1, 900)]
    q, ks, vs, caches = make_seqs(shapes, H, Hkv, 8, "cuda")
    batch = PagedBatch(caches, [64, 1])
    o, lse = torch.zeros(65, H * HD, dtype=BF, device="cuda"), torch.zeros(65, H, device="cuda")
    mass = [torch.zeros(Hkv, p, device="cuda") for _, p in shapes]
    into = PagedKVCache(1, Hkv, HD, keep, device="cuda")
    kept = torch.zeros(1, Hkv, keep, dtype=torch.int32, device="cuda")
    ws = torch.zeros(max(_lib.attn_window_workspace_bytes(65, H),
                         _lib.attn_key_mass_workspace_bytes(2400, Hkv)), dtype=torch.uint8,
                     device="cuda")
    left = torch.zeros(1, Hkv, keep, device="cuda")

    def step():
        _lib.attn_window(q, batch, 0, H, HD ** -0.5, o, ws, lse=lse, block=32, window=400, sinks=4)
        _lib.attn_key_mass(q, lse, batch, 0, H, HD ** -0.5, mass, ws, block=32, window=400, sinks=4)
        caches[0].evict(mass[0][None], keep, sinks=4, recent=200, into=into, kept=kept,
                        mass_out=left)

    outs = (o, lse, mass[0], mass[1], kept, left, into.k_pages, into.v_pages)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    g = torch.Generator(device="cuda").manual_seed(3)
    for rep in range(4):
        q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
        for t in outs:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        for t in outs:
            t.zero_()
        step()
        torch.cuda.synchronize()
        for a, b in zip(got, outs):
            assert torch.equal(a.view(torch.int32) if a.dtype == torch.float32 else a.view(torch.int16)
                               if a.dtype == BF else a,
                               b.view(torch.int32) if b.dtype == torch.float32 else b.view(torch.int16)
                               if b.dtype == BF else b), rep
        _work_between()


def test_two_streams_two_workspaces():
    """Two calls at once on streams of their own."""
    H, Hkv = 32, 8
    sets = [make_seqs([(200, 3000)], H, Hkv, 20 + i, "cuda") for i in range(2)]
    refs = [run_window(_lib, q, c, [200], H, 1, 0, 0) for q, _, _, c in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    outs = []
    for (q, _, _, c), st in zip(sets, streams):
        o = torch.zeros(200, H * HD, dtype=BF, device="cuda")
        ws = torch.zeros(_lib.attn_window_workspace_bytes(200, H), dtype=torch.uint8, device="cuda")
        outs.append((o, ws, PagedBatch(c, [200])))
    torch.cuda.synchronize()
    for _ in range(3):
        for (q, _, _, c), st, (o, ws, batch) in zip(sets, streams, outs):
            _lib.attn_window(q, batch, 0, H, HD ** -0.5, o, ws, stream=st)
    torch.cuda.synchronize()
    for (o, _, _), (ref, _) in zip(outs, refs):
        assert torch.equal(o.view(200, H, HD), ref)


def test_long_offsets():
    """A cache whose element offsets pass 2^32: pages far apart."""
    H, Hkv, P = 8, 2, 200
    q, ks, vs, caches = make_seqs([(3, P)], H, Hkv, 12, "cuda")
    page, pages = 128, 70000           # 70000 pages of 128 * 2 * 128 elements: 4.6 G elements
    c = object.__new__(PagedKVCache)
    small = PagedKVCache(1, Hkv, HD, 2 * page, page_size=page, device="cuda")
    c.__dict__.update(small.__dict__)
    pool = torch.empty(1, pages, Hkv, page, HD, dtype=BF, device="cuda")
    c.k_pages = c.v_pages = pool
    c.num_pages, c.capacity = pages, pages * page
    c.page_table = torch.tensor([pages - 1, pages - 3], dtype=torch.int32, device="cuda")
    for i, at in enumerate((pages - 1, pages - 3)):
        n = min(page, P - i * page)
        pool[0, at, :, :n] = ks[0][:, i * page:i * page + n]
    c.advance(P)
    o, lse = run_window(_lib, q, [c], [3], H)
    ro, rl, tol, tol_l = plain_attention(q[:3], ks[0], ks[0])
    assert torch.all((o.double() - ro).abs() <= tol)
    out = [torch.zeros(Hkv, P, device="cuda")]
    ws = torch.zeros(_lib.attn_key_mass_workspace_bytes(P, Hkv), dtype=torch.uint8, device="cuda")
    _lib.attn_key_mass(q, lse, PagedBatch([c], [3]), 0, H, HD ** -0.5, out, ws)
    ref, tm = plain_mass(q[:3], lse, ks[0])
    assert torch.all((out[0].double() - ref).abs() <= tm + 2.0 ** -23 * ref + 1e-30)
    # (K and V share the pool here: moving either moves both alike)
    kept = c.evict(out[0][None], 64, sinks=2, recent=8)
    at = kept[0].long()[..., None].expand(-1, -1, HD)
    assert torch.equal(pool[0, pages - 1, :, :64], torch.gather(ks[0], 1, at))


# ---- through the engine ----------------------------------------------------------------------


@pytest.mark.parametrize("shape,causal", [(SHAPE_G2, False), (SHAPE_N8, True)])
def test_prompt_under_a_window(shape, causal, monkeypatch):
    """append_prompt with a window and key_mass: every layer's attention and mass against
    the plain forms on that layer's own queries and cache; eviction; the prompt goes on; the
    verify step takes its positions from behind the evicted keys."""
    build = build_nld if causal else build_qwen2
    model = to_gpu_model(build(shape, 3, device="cpu", dtype=BF))
    eng = FoldedVerifyEngine(model)
    L, H, Hkv = eng.L, eng.H, eng.Hkv
    G = H // Hkv
    cache = PagedKVCache(L, Hkv, HD, 1024, device="cuda", page_order="shuffled", seed=4)
    mass = torch.zeros(L, Hkv, 1024, device="cuda")
    mask = dict(block=1 if causal else 32, window=100, sinks=4)
    calls = []
    real, real_mass = _lib.attn_window, _lib.attn_key_mass

    def attn(q, batch, li, H_, scaling, o, ws, lse=None, **kw):
        assert kw == mask
        real(q, batch, li, H_, scaling, o, ws, lse=lse, **kw)
        n, c = batch.num_rows, batch.caches[0]
        keep_len, c.length = c.length, c.length + n
        k, v = (x[0] for x in c[li])
        c.length = keep_len
        ro, rl, tol, tol_l = plain_attention(q[:n].view(n, H, HD), k, v, scaling=scaling, **kw)
        assert torch.all((o[:n].view(n, H, HD).double() - ro).abs() <= tol)
        assert torch.all((lse.double() - rl).abs() <= tol_l)
        calls.append((li, n, c.length))

    def key_mass(q, lse, batch, li, H_, scaling, out, ws, mass_in=None, **kw):
        n, c = batch.num_rows, batch.caches[0]
        P = c.length + n
        was = out[0][:, :P].clone()
        real_mass(q, lse, batch, li, H_, scaling, out, ws, mass_in=mass_in, **kw)
        keep_len, c.length = c.length, P
        k = c[li][0][0]
        c.length = keep_len
        ref, tol = plain_mass(q[:n].view(n, H, HD), lse, k, scaling=scaling, **kw)
        d = (out[0][:, :P].double() - was.double() - ref).abs()
        assert torch.all(d <= tol + 2.0 ** -22 * (ref + was))

    monkeypatch.setattr(_lib, "attn_window", attn)
    monkeypatch.setattr(_lib, "attn_key_mass", key_mass)
    g = torch.Generator().manual_seed(2)
    toks = torch.randint(0, shape.vocab - 1, (1, 333), generator=g).cuda()
    logits = eng.append_prompt(toks, cache, 32, causal=causal, window=100, sinks=4, key_mass=mass)
    assert logits.shape == (1, 333, eng.V) and torch.all(logits.isfinite())
    assert calls == [(li, 333, 0) for li in range(L)]
    # every row's weights sum to one
    assert torch.all((mass.sum(-1) - 333 * G).abs() < 0.05)
    kept = cache.evict(mass, 120, sinks=4, recent=64)
    assert torch.all(kept[..., :4].cpu() == torch.arange(4))
    assert torch.all(kept[..., -64:].cpu() == torch.arange(333 - 64, 333))
    assert (cache.length, cache.position) == (120, 333)
    eng.append_prompt(toks[:, :32], cache, 32, causal=causal, window=100, sinks=4, key_mass=mass)
    assert (cache.length, cache.position) == (152, 365) and len(calls) == 2 * L

    # the verify step: the block's RoPE at positions 365.., whatever is left in the cache
    full = PagedKVCache(L, Hkv, HD, 1024, device="cuda")
    full.advance(365)
    blk = torch.randint(0, shape.vocab - 1, (2, 32), generator=g)
    blk[1, :] = blk[0, :]
    blk[1, 3] = (blk[0, 3] + 1) % (shape.vocab - 1)
    t1, t2 = [], []
    a = eng.forward(blk.cuda(), cache, 0.1, trace=t1)
    eng.forward(blk.cuda(), full, 0.1, trace=t2)
    cnt = int(t1[0]["count"])
    rows = t1[0]["rows"][:cnt].long()
    assert torch.equal(t1[0]["q"][rows], t2[0]["q"][rows])
    assert torch.equal(t1[0]["kv"][rows], t2[0]["kv"][rows])
    for _ in range(3):     # the captured step takes the same positions
        b = eng.forward(blk.cuda(), cache, 0.1)
        assert torch.equal(a, b)
        _work_between()
    # and a batched step
    c = eng.forward_batched([blk.cuda(), blk.cuda()], [cache, full], 0.1)
    assert torch.allclose(c[0].float(), a.float(), atol=0.05, rtol=0.05)
    assert torch.all(a.isfinite())


def test_append_refusals():
    model = to_gpu_model(build_qwen2(SHAPE_G2, 3, device="cpu", dtype=BF))
    eng = FoldedVerifyEngine(model)
    cache = PagedKVCache(eng.L, eng.Hkv, HD, 128, device="cuda")
    toks = torch.zeros(1, 64, dtype=torch.long, device="cuda")
    for kw in (dict(window=-1), dict(sinks=4), dict(window=10, sinks=-1),
               dict(key_mass=torch.zeros(eng.L, eng.Hkv, 63, device="cuda")),
               dict(key_mass=torch.zeros(eng.L, eng.Hkv + 1, 64, device="cuda")),
               dict(key_mass=torch.zeros(eng.L, eng.Hkv, 64, device="cuda").double())):
        with pytest.raises(ValueError):
            eng.append_blocks(toks, cache, 32, **kw)
    with pytest.raises(ValueError):
        eng.append_prompt(torch.zeros(1, 200, dtype=torch.long, device="cuda"), cache, 32, window=10)
    with pytest.raises(ValueError):
        _lib.attn_window(torch.zeros(4, 512, dtype=BF), PagedBatch([cache], [0]), 0, 4, 0.1,
                         torch.zeros(4, 512, dtype=BF), torch.zeros(64, dtype=torch.uint8))
    assert cache.length == 0
