"""sf_attn_window, sf_attn_key_mass and sf_kv_evict: the kernels' own sources on the CPU
simulator against 64-bit forms, and the refusals of the library and its wrappers."""

import ctypes
import math

import pytest
import torch

from specfold_amd import _lib
from specfold_amd.kv_cache import ContiguousMirror, PagedBatch, PagedKVCache
from tests.bounded_cache import (BF, HD, check_evict, check_mass, check_window, make_seqs,
                                 plain_attention, plain_mass, run_window, seen)
from tests.simlib import build_sim_library, compiler, use_sim_library


@pytest.fixture(scope="module")
def sim(tmp_path_factory):
    if compiler() is None:
        pytest.skip("no clang++ (the simulator needs clang's vector extensions)")
    with use_sim_library(build_sim_library(tmp_path_factory.mktemp("simlib"))) as lib:
        yield lib


# (n, P) of each sequence, H, Hkv, block, window, sinks, page
WINDOW = [
    ([(1, 1)], 4, 2, 1, 0, 0, 16),                     # the first token of all
    ([(1, 200)], 7, 1, 1, 0, 0, 16),                   # one token, odd head group
    ([(1, 200)], 8, 2, 1, 50, 3, 16),                  # one token, window and sinks
    ([(1, 333), (1, 17), (1, 64)], 8, 2, 1, 100, 4, 32),
    ([(0, 0), (2, 70), (0, 40), (1, 1)], 4, 2, 1, 0, 0, 16),   # empty sequences
    ([(33, 150)], 4, 2, 32, 0, 0, 16),                 # a short last block
    ([(40, 40), (5, 90)], 4, 1, 8, 0, 0, 64),
    ([(70, 220)], 6, 2, 1, 0, 0, 16),
    ([(70, 220)], 6, 2, 1, 1, 0, 16),                  # a row sees itself alone
    ([(70, 220)], 6, 2, 1, 40, 0, 16),
    ([(70, 400)], 6, 2, 32, 64, 5, 16),
    ([(100, 300)], 4, 2, 16, 33, 70, 128),             # sinks past a chunk
    ([(64, 64)], 4, 4, 64, 500, 2, 16),                # a window wider than all
    ([(20, 60)], 16, 1, 4, 7, 1, 16),                  # 16 heads a kv head
    ([(130, 131), (67, 300)], 5, 1, 32, 100, 2, 16),
    ([(1, 400), (2, 520), (1, 30), (0, 9)], 8, 2, 1, 0, 0, 16),   # few queries, more stages
    ([(3, 700)], 4, 2, 2, 350, 20, 64),
]


@pytest.mark.parametrize("shapes,H,Hkv,block,window,sinks,page", WINDOW)
def test_window(sim, shapes, H, Hkv, block, window, sinks, page):
    check_window(sim, shapes, H, Hkv, block, window, sinks, "cpu", seed=len(shapes) + window,
                 page=page)


def test_window_large_scores(sim):
    """Scores far apart: the running maximum moves from chunk to chunk."""
    check_window(sim, [(40, 300)], 4, 2, 8, 0, 0, "cpu", std=6.0)


def test_window_contiguous(sim):
    """A cache without a page table beside the same keys in pages."""
    q, ks, vs, caches = make_seqs([(9, 130)], 4, 2, 3, "cpu")
    mirror = ContiguousMirror(1, 2, HD, 200, device="cpu")
    mirror.sync([(ks[0][None], vs[0][None])])
    o, lse = run_window(sim, q, caches, [9], 4, 4, 60, 2)
    o2, lse2 = run_window(sim, q, [mirror], [9], 4, 4, 60, 2)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


# a key that some rows do not see: behind their block, in front of their window, in a chunk
# that others of the tile see
@pytest.mark.parametrize("n,P,block,window,sinks,at", [
    (64, 64, 32, 0, 0, 40), (70, 220, 1, 0, 0, 200), (70, 220, 1, 30, 0, 155),
    (70, 400, 32, 64, 5, 300), (40, 300, 8, 100, 3, 2), (2, 130, 1, 0, 0, 129),
    (2, 400, 1, 0, 0, 399), (3, 400, 1, 300, 4, 99)])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_hidden_key_not_finite(sim, n, P, block, window, sinks, at, bad):
    H, Hkv = 4, 2
    q, ks, vs, caches = make_seqs([(n, P)], H, Hkv, n + P, "cpu")
    kz, vz = ks[0].clone(), vs[0].clone()
    k, v = ks[0].clone(), vs[0].clone()
    v[1, at, [3, 64]], vz[1, at, [3, 64]] = bad, 0
    if bad != bad:
        k[1, at, 5], kz[1, at, 5] = bad, 0
    c = PagedKVCache(1, Hkv, HD, P, device="cpu", page_order="shuffled", seed=2)
    c.load_dense([(k[None], v[None])])
    o, lse = run_window(sim, q, [c], [n], H, block, window, sinks)
    ro, rl, tol, tol_l = plain_attention(q[:n], kz, vz, block, window, sinks)
    see = seen(n, P, block, window, sinks)[:, at]
    heads = torch.arange(H) >= H // Hkv
    ok = (o.double() - ro).abs() <= tol
    assert torch.all(ok[~see]) and torch.all(ok[:, ~heads])
    okl = (lse.double() - rl).abs() <= tol_l
    assert torch.all(okl[~see]) and torch.all(okl[:, ~heads])
    hit = o[see][:, heads]
    assert not torch.any(hit[..., [3, 64]].isfinite())
    if bad == bad:
        ok[..., [3, 64]] = True
        assert torch.all(ok)
    else:
        assert torch.all(lse[see][:, heads].isnan())


MASS = [
    ([(1, 1)], 4, 2, 1, 0, 0, 16),
    ([(1, 200)], 7, 1, 1, 0, 0, 16),
    ([(1, 333), (0, 40), (1, 64)], 8, 2, 1, 100, 4, 32),
    ([(33, 150)], 4, 2, 32, 0, 0, 16),
    ([(70, 400), (3, 500)], 6, 2, 32, 64, 5, 16),
    ([(20, 60)], 16, 1, 4, 7, 1, 64),
    ([(130, 300)], 5, 1, 1, 0, 0, 16),
]


@pytest.mark.parametrize("shapes,H,Hkv,block,window,sinks,page", MASS)
@pytest.mark.parametrize("how", ["fresh", "add", "inplace"])
def test_mass(sim, shapes, H, Hkv, block, window, sinks, page, how):
    check_mass(sim, shapes, H, Hkv, block, window, sinks, "cpu", page=page,
               decay=0.75 if how == "inplace" else 1.0, inplace=how == "inplace",
               fresh=how == "fresh")


def test_mass_hidden_key_not_finite(sim):
    """A NaN key makes its own sum NaN where a row sees it and no other."""
    q, ks, vs, caches = make_seqs([(6, 100)], 4, 2, 3, "cpu")
    caches[0].k_pages[0, caches[0].page_table[99 // 16], 1, 99 % 16, 7] = math.nan
    caches[0].k_pages[0, caches[0].page_table[10 // 16], 0, 10 % 16, 7] = math.nan
    lse = plain_attention(q, ks[0], vs[0], 1, 20, 4)[1].float()
    out = [torch.zeros(2, 100)]
    ws = torch.zeros(sim.attn_key_mass_workspace_bytes(100, 2), dtype=torch.uint8)
    sim.attn_key_mass(q, lse, PagedBatch(caches, [6]), 0, 4, HD ** -0.5, out, ws, window=20, sinks=4)
    ref, tol = plain_mass(q, lse, ks[0], 1, 20, 4)
    bad = out[0].isnan()
    assert bad[1, 99] and bad.sum() == 1
    assert torch.all(((out[0].double() - ref).abs() <= tol + 2.0 ** -23 * ref + 1e-30)[~bad])


EVICT = [
    # L, Hkv, length, keep, sinks, recent
    (1, 1, 1, 1, 0, 0), (2, 3, 40, 40, 4, 8), (1, 2, 40, 1, 0, 0), (1, 2, 40, 1, 1, 0),
    (1, 2, 40, 1, 0, 1), (2, 2, 301, 150, 4, 32), (1, 2, 301, 140, 70, 70), (1, 1, 700, 300, 0, 0),
    (1, 1, 5000, 600, 4, 64), (1, 2, 130, 129, 0, 0), (1, 1, 1100, 1024, 0, 5),
]


@pytest.mark.parametrize("case", EVICT)
@pytest.mark.parametrize("into", [False, True])
def test_evict(sim, case, into):
    check_evict(*case, "cpu", into, page2=64 if case[2] % 2 else None)


@pytest.mark.parametrize("kind", ["equal", "zeros", "nan", "inf", "negative"])
def test_evict_orders(sim, kind):
    """Equal masses keep the lower slots; -0 is 0; NaN above inf above all numbers."""
    g = torch.Generator().manual_seed(4)
    m = torch.randn(1, 2, 90, generator=g)
    if kind == "equal":
        m.fill_(0.25)
    elif kind == "zeros":
        m = torch.where(m > 0, 0.0, -0.0)
    elif kind == "nan":
        m[:, :, ::7] = math.nan
        m[:, 1, 3::7] = -math.nan
        m[:, :, 5::9] = math.inf
    elif kind == "inf":
        m[:, :, ::3] = math.inf
        m[:, :, 1::3] = -math.inf
    for into in (False, True):
        check_evict(1, 2, 90, 30, 2, 5, "cpu", into, mass=m.clone())


def test_evicted_cache_goes_on(sim):
    """Eviction, append, attention and mass over what is left, eviction again."""
    H, Hkv = 4, 2
    g = torch.Generator().manual_seed(9)
    c = PagedKVCache(1, Hkv, HD, 160, device="cpu", page_order="shuffled", seed=2)
    k, v = (torch.randn(1, Hkv, 130, HD, generator=g).to(BF) for _ in range(2))
    c.load_dense([(k, v)])
    mass = torch.rand(1, Hkv, 160, generator=g)
    for step in range(2):
        P = c.length
        kept = c.evict(mass, 64, sinks=4, recent=16)
        at = kept[0].long()[..., None].expand(-1, -1, HD)
        k, v = (torch.gather(x[0], 1, at)[None] for x in (k, v))
        assert c.length == 64 and c.position == 130 + 32 * step
        new = torch.randn(32, 2, Hkv, HD, generator=g).to(BF)
        c.append_rows(0, new.view(32, -1), 0, 32)
        k, v = (torch.cat([x, new[:, i].transpose(0, 1)[None]], 2) for i, x in enumerate((k, v)))
        q = torch.randn(32, H, HD, generator=g).to(BF)
        batch = PagedBatch([c], [32], ahead=True)
        o, lse = torch.empty(32, H * HD, dtype=BF), torch.empty(32, H)
        ws = torch.zeros(sim.attn_window_workspace_bytes(32, H), dtype=torch.uint8)
        sim.attn_window(q, batch, 0, H, HD ** -0.5, o, ws, lse=lse, block=32)
        wm = torch.zeros(sim.attn_key_mass_workspace_bytes(96, Hkv), dtype=torch.uint8)
        before = mass.clone()
        sim.attn_key_mass(q, lse, batch, 0, H, HD ** -0.5, [mass[0]], wm, mass_in=[mass[0]],
                          block=32)
        c.advance(32)
        ro, rl, tol, tol_l = plain_attention(q, k[0], v[0], 32)
        assert torch.all((o.view(32, H, HD).double() - ro).abs() <= tol)
        assert torch.all((lse.double() - rl).abs() <= tol_l)
        got, tm = plain_mass(q, lse, k[0], 32)
        ref = before[0, :, :96].double() + got
        assert torch.all((mass[0, :, :96].double() - ref).abs() <= tm + 2.0 ** -22 * ref)
        assert P == (130 if step == 0 else 96)
        # every row's weights sum to one
        assert abs(float((mass[0, :, :96] - before[0, :, :96]).sum()) - 32 * H) < 1e-2


# ---- refusals: nothing is launched (the pointers are never read) -----------------------------


def _call(lib, what, **over):
    p = [ctypes.c_void_p(4096 * (i + 1)) for i in range(8)]
    a = dict(q=p[0], n_seqs=1, page_size=16, block=1, window=0, sinks=0, H=4, Hkv=2, hd=128,
             o=p[3], lse=p[4], ws=p[5], ws_bytes=1 << 30, decay=1.0)
    s = dict(k=4096, v=8192, page_table=256, mass_in=None, mass_out=512, page_stride=4096,
             head_stride=2048, mass_in_stride=0, mass_out_stride=64, length=64, rows=8, pages=4,
             reserved=0)
    for key, val in over.items():
        (s if key in s else a)[key] = val
    arr = (_lib.KVSeq * max(1, a["n_seqs"]))()
    for e in arr:
        for key, val in s.items():
            setattr(e, key, val)
    seqs = arr if over.get("seqs", 1) else None
    if what == "window":
        return lib.sf_attn_window(a["q"], seqs, a["n_seqs"], a["page_size"], a["block"],
                                  a["window"], a["sinks"], a["H"], a["Hkv"], a["hd"], 0.1, a["o"],
                                  a["lse"], a["ws"], a["ws_bytes"], None)
    return lib.sf_attn_key_mass(a["q"], a["lse"], seqs, a["n_seqs"], a["page_size"], a["block"],
                                a["window"], a["sinks"], a["H"], a["Hkv"], a["hd"], 0.1,
                                a["decay"], a["ws"], a["ws_bytes"], None)


SHAPE, ARG, WORKSPACE = 1, 2, 3


@pytest.mark.parametrize("what", ["window", "mass"])
@pytest.mark.parametrize("over,code", [
    (dict(seqs=0), ARG), (dict(q=None), ARG), (dict(ws=None), ARG),
    (dict(q=ctypes.c_void_p(4104)), ARG), (dict(ws=ctypes.c_void_p(4100)), ARG),
    (dict(k=0), ARG), (dict(k=4104), ARG), (dict(reserved=1), ARG),
    (dict(n_seqs=0), SHAPE), (dict(n_seqs=33), SHAPE), (dict(hd=64), SHAPE), (dict(H=5), SHAPE),
    (dict(H=34), SHAPE), (dict(Hkv=0), SHAPE), (dict(block=0), SHAPE), (dict(window=-1), SHAPE),
    (dict(sinks=-1), SHAPE), (dict(page_size=8), SHAPE), (dict(page_size=48), SHAPE),
    (dict(page_size=256), SHAPE), (dict(pages=0), SHAPE), (dict(rows=-1), SHAPE),
    (dict(rows=65), SHAPE), (dict(length=-1), SHAPE), (dict(length=32769), SHAPE),
    (dict(page_stride=4100), SHAPE), (dict(head_stride=2044), SHAPE),
    (dict(page_table=None, head_stride=128 * 63), SHAPE), (dict(ws_bytes=0), WORKSPACE)])
def test_refusals(what, over, code):
    assert _call(_lib.load(), what, **over) == code


@pytest.mark.parametrize("what,over,code", [
    ("window", dict(v=0), ARG), ("window", dict(o=None), ARG),
    ("window", dict(o=ctypes.c_void_p(4104)), ARG), ("mass", dict(lse=None), ARG),
    ("mass", dict(mass_out=None), ARG), ("mass", dict(mass_out_stride=63), SHAPE),
    ("mass", dict(mass_in=1024, mass_in_stride=63), SHAPE),
    ("mass", dict(mass_in=512, mass_in_stride=65), ARG), ("mass", dict(decay=-0.1), ARG),
    ("mass", dict(decay=1.5), ARG), ("mass", dict(decay=math.nan), ARG)])
def test_refusals_of_one(what, over, code):
    assert _call(_lib.load(), what, **over) == code


def test_nothing_to_do():
    """No rows: fine without pointers."""
    lib = _lib.load()
    assert _call(lib, "window", rows=0, q=None, o=None, ws=None) == 0
    assert _call(lib, "mass", rows=0, length=0, q=None, lse=None, ws=None) == 0


def _evict(lib, **over):
    a = dict(mass=4096, layers=1, Hkv=2, hd=128, P=64, sinks=2, recent=4, keep=32, kept=8192,
             mass_out=None, ml=128, mh=64, oml=0, omh=0, same=True)
    p = dict(k=4096, v=8192, page_table=512, layer_stride=16384, page_stride=4096,
             head_stride=2048, page_size=16, pages=4)
    t = dict(p)
    for key, val in over.items():
        if key.startswith("to_"):
            t[key[3:]] = val
        elif key in p:
            p[key] = val
        else:
            a[key] = val
    f, to = _lib.KVPages(**p), _lib.KVPages(**t)
    return lib.sf_kv_evict(a["mass"], a["ml"], a["mh"], a["layers"], a["Hkv"], a["hd"], a["P"],
                           a["sinks"], a["recent"], a["keep"], ctypes.byref(f), ctypes.byref(to),
                           a["kept"], a["mass_out"], a["oml"], a["omh"], None, None, 0, None)


@pytest.mark.parametrize("over,code", [
    (dict(mass=None), ARG), (dict(kept=None), ARG), (dict(k=None), ARG), (dict(to_v=None), ARG),
    (dict(page_table=None), ARG), (dict(to_k=4104), ARG), (dict(hd=64), SHAPE),
    (dict(layers=0), SHAPE), (dict(Hkv=0), SHAPE), (dict(P=0), SHAPE), (dict(P=32769), SHAPE),
    (dict(keep=0), SHAPE), (dict(keep=65), SHAPE), (dict(sinks=-1), SHAPE),
    (dict(recent=-1), SHAPE), (dict(sinks=30, recent=3), SHAPE), (dict(sinks=33), SHAPE),
    (dict(page_size=24), SHAPE), (dict(to_page_size=8), SHAPE), (dict(pages=3), SHAPE),
    (dict(to_pages=1), SHAPE), (dict(page_stride=4), SHAPE), (dict(to_layer_stride=7), SHAPE),
    (dict(to_v=4096 * 5), ARG), (dict(to_head_stride=4096), ARG), (dict(to_page_size=32), ARG),
    (dict(mass_out=4096, oml=128, omh=63), ARG),
    # rows of mass_out over each other
    (dict(mass_out=16384, oml=64, omh=31), SHAPE), (dict(mass_out=4096, mh=63, omh=63, oml=128), SHAPE),
    (dict(mass_out=16384, layers=3, oml=63, omh=32), SHAPE),
    (dict(mass_out=16384, layers=3, oml=32, omh=95), SHAPE),
    (dict(mass_out=16384, layers=3, oml=31, omh=96), SHAPE),
    (dict(mass_out=16384, layers=3, Hkv=1, oml=0), SHAPE)])
def test_evict_refusals(over, code):
    assert _evict(_lib.load(), **over) == code


def test_wrapper_refusals(sim):
    q, ks, vs, caches = make_seqs([(3, 20)], 4, 2, 1, "cpu")
    o, ws = torch.empty(3, 512, dtype=BF), torch.empty(1 << 23, dtype=torch.uint8)
    batch = PagedBatch(caches, [3])
    with pytest.raises(TypeError):
        sim.attn_window(q.float(), batch, 0, 4, 0.1, o, ws)
    with pytest.raises(ValueError):
        sim.attn_window(q, batch, 0, 8, 0.1, o, ws)                  # q too small for 8 heads
    with pytest.raises(ValueError):
        sim.attn_window(q.transpose(0, 1), batch, 0, 4, 0.1, o, ws)  # not contiguous
    with pytest.raises(_lib.SpecFoldKernelError):
        sim.attn_window(q, PagedBatch(caches, [3]), 0, 4, 0.1, o, ws, window=-3)
    with pytest.raises(ValueError):
        PagedBatch(caches, [3, 1])
    with pytest.raises(ValueError):
        PagedBatch([], [])
    with pytest.raises(ValueError):
        PagedBatch(caches, [-1])
    with pytest.raises(TypeError):
        PagedBatch([object.__new__(type("C", (), dict(Hkv=2, hd=128, length_dev=torch.zeros(1))))],
                   [1])
    with pytest.raises(ValueError):
        PagedBatch([caches[0], PagedKVCache(1, 2, HD, 64, page_size=32, device="cpu")], [1, 1])
    with pytest.raises(_lib.SpecFoldKernelError):     # more rows than keys
        sim.attn_window(torch.zeros(21, 512, dtype=BF), PagedBatch(caches, [21]), 0, 4, 0.1,
                        torch.empty(21, 512, dtype=BF), ws)
    lse = torch.zeros(3, 4)
    for mass in ([torch.zeros(2, 19)], [torch.zeros(3, 20)], [torch.zeros(20, 2).t()],
                 [torch.zeros(2, 20).double()], []):
        with pytest.raises(ValueError):
            sim.attn_key_mass(q, lse, batch, 0, 4, 0.1, mass, ws)
    c = caches[0]
    mass = torch.zeros(1, 2, 20)
    for kw in (dict(keep=0), dict(keep=21), dict(keep=5, sinks=3, recent=3), dict(keep=5, sinks=-1),
               dict(keep=5, into=c)):
        with pytest.raises(ValueError):
            c.evict(mass, **kw)
    with pytest.raises(ValueError):
        c.evict(mass[..., :19], keep=5)
    with pytest.raises(ValueError):
        c.evict(mass, keep=18, into=PagedKVCache(1, 2, HD, 16, device="cpu"))
    with pytest.raises(ValueError):
        c.evict(mass, keep=5, into=PagedKVCache(2, 2, HD, 16, device="cpu"))
    assert c.length == 20 and c.position == 20


def test_bad_pages_stay_inside(sim):
    """Page ids outside the pool are read as page 0 and never written."""
    q, ks, vs, caches = make_seqs([(3, 40)], 4, 2, 1, "cpu")
    c = caches[0]
    c.page_table[0], c.page_table[1] = -1, 1 << 30
    o, lse = run_window(sim, q, caches, [3], 4)
    out = [torch.zeros(2, 40)]
    ws = torch.zeros(sim.attn_key_mass_workspace_bytes(40, 2), dtype=torch.uint8)
    sim.attn_key_mass(q, lse, PagedBatch(caches, [3]), 0, 4, HD ** -0.5, out, ws)
    before = c.k_pages.clone()
    mapped = c.page_table.tolist()
    c.evict(torch.rand(1, 2, 40), 30)
    others = [pg for pg in range(c.num_pages) if pg not in mapped]
    assert len(others) == 2
    assert torch.equal(c.k_pages[:, others].view(torch.int16), before[:, others].view(torch.int16))


@pytest.mark.parametrize("what", ["window", "mass"])
@pytest.mark.parametrize("scaling", [0.0, -0.1, math.inf, math.nan])
def test_scaling_refused(sim, what, scaling):
    q, ks, vs, caches = make_seqs([(3, 20)], 4, 2, 1, "cpu")
    ws = torch.empty(1 << 23, dtype=torch.uint8)
    batch = PagedBatch(caches, [3])
    with pytest.raises(_lib.SpecFoldKernelError):
        if what == "window":
            sim.attn_window(q, batch, 0, 4, scaling, torch.empty(3, 512, dtype=BF), ws)
        else:
            sim.attn_key_mass(q, torch.zeros(3, 4), batch, 0, 4, scaling, [torch.zeros(2, 20)], ws)


def test_too_many_heads_refused():
    for what in ("window", "mass"):
        assert _call(_lib.load(), what, H=272, Hkv=17, mass_out_stride=64) == SHAPE


def test_shared_mass_refused(sim):
    """Two sequences that write one array, or of which one reads what the other writes."""
    q, ks, vs, caches = make_seqs([(1, 20), (2, 24)], 4, 2, 1, "cpu")
    batch, lse = PagedBatch(caches, [1, 2]), torch.zeros(3, 4)
    ws = torch.empty(sim.attn_key_mass_workspace_bytes(44, 2), dtype=torch.uint8)
    a, b, c = (torch.zeros(2, 24) for _ in range(3))
    for out, had in (([a, a], None), ([a, b], [b, c]), ([a, b], [c, a])):
        with pytest.raises(_lib.SpecFoldKernelError):
            sim.attn_key_mass(q, lse, batch, 0, 4, 0.1, out, ws, mass_in=had)
    sim.attn_key_mass(q, lse, batch, 0, 4, 0.1, [a, b], ws, mass_in=[c, c])   # reading one is fine


def test_batch_follows_its_caches(sim):
    """A batch that was used before a cache got other buffers (and lengths) reads those; one
    cache twice in a batch is two sequences."""
    q, ks, vs, caches = make_seqs([(2, 40)], 4, 2, 1, "cpu")
    batch, ws = PagedBatch(caches, [2]), torch.empty(1 << 23, dtype=torch.uint8)
    outs = [torch.empty(2, 512, dtype=BF) for _ in range(3)]
    sim.attn_window(q, batch, 0, 4, HD ** -0.5, outs[0], ws)
    caches[0].v_pages.neg_()
    sim.attn_window(q, batch, 0, 4, HD ** -0.5, outs[1], ws)
    assert torch.equal(outs[1], -outs[0])
    caches[0].v_pages = -caches[0].v_pages
    sim.attn_window(q, batch, 0, 4, HD ** -0.5, outs[2], ws)
    assert torch.equal(outs[2], outs[0])
    twice = torch.empty(4, 512, dtype=BF)
    sim.attn_window(torch.cat([q, q]), PagedBatch(caches * 2, [2, 2]), 0, 4, HD ** -0.5, twice, ws)
    assert torch.equal(twice, torch.cat([outs[0], outs[0]]))
    with pytest.raises(ValueError):
        PagedBatch([caches[0], PagedKVCache(1, 2, 64, 64, page_size=16, device="cpu")], [1, 1])
    # a call refused for lengths past the capacity leaves nothing of them behind
    c = caches[0]
    c.length = 38
    ahead = PagedBatch([c], [2], ahead=True)
    sim.attn_window(q, ahead, 0, 4, HD ** -0.5, outs[1], ws)
    c.length = c.capacity
    with pytest.raises(ValueError):
        sim.attn_window(q, ahead, 0, 4, HD ** -0.5, outs[1], ws)
    c.length = 38
    outs[1].zero_()
    sim.attn_window(q, ahead, 0, 4, HD ** -0.5, outs[1], ws)
    assert torch.equal(outs[1], outs[0])


def test_mass_of_a_row_without_a_number(sim):
    """A row whose lse is NaN or -inf reaches the keys it sees, and no other."""
    q, ks, vs, caches = make_seqs([(40, 100)], 4, 2, 1, "cpu")
    ws = torch.empty(sim.attn_key_mass_workspace_bytes(100, 2), dtype=torch.uint8)
    lse = torch.zeros(40, 4)
    lse[7] = float("nan")
    lse[9, 0] = -math.inf
    out = [torch.zeros(2, 100)]
    sim.attn_key_mass(q, lse, PagedBatch(caches, [40]), 0, 4, HD ** -0.5, out, ws)
    assert out[0][:, :68].isnan().all() and out[0][1, 68:].isfinite().all()
    assert (out[0][0, 68:70] == math.inf).all() and out[0][0, 70:].isfinite().all()


def test_extreme_masks(sim):
    """Windows, sinks and blocks as large as an int holds are no mask at all."""
    big = 2 ** 31 - 1
    q, ks, vs, caches = make_seqs([(40, 100)], 4, 2, 1, "cpu")
    ref = run_window(sim, q, caches, [40], 4, 1, 0, 0)
    for window, sinks in ((big, 0), (big, big), (1, big), (0, big)):
        got = run_window(sim, q, caches, [40], 4, 1, window, sinks)
        assert torch.equal(ref[0], got[0]) and torch.equal(ref[1], got[1])
    ref = run_window(sim, q, caches, [40], 4, 40, 0, 0)
    got = run_window(sim, q, caches, [40], 4, big, 0, 0)
    assert torch.equal(ref[0], got[0]) and torch.equal(ref[1], got[1])
    for window, sinks, block in ((big, 0, 1), (1, big, 1), (0, big, big)):
        ws = torch.zeros(sim.attn_key_mass_workspace_bytes(100, 2), dtype=torch.uint8)
        outs = []
        for kw in (dict(block=block), dict(block=block, window=window, sinks=sinks)):
            out = [torch.zeros(2, 100)]
            sim.attn_key_mass(q, ref[1].contiguous(), PagedBatch(caches, [40]), 0, 4, HD ** -0.5,
                              out, ws, **kw)
            outs.append(out[0])
        assert torch.equal(*outs)
