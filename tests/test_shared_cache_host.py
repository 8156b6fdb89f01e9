"""Host side of the operators around a shared cache: pages and their holders, refusals, the gradient formulas against
differences.  No GPU."""
import random

import pytest
import torch

import shared_cache_ref as R


def _pool(P=4, per_slab=3):
    from loquetier_b200 import kvcache
    return kvcache.KvPool(1, 1, 8, P, torch.float32, "cpu", pages_per_slab=per_slab)


@pytest.fixture
def cpu_copies(monkeypatch):
    """Page copies on host memory in place of the kernel's."""
    from loquetier_b200 import kvcache

    def tables(device, dst, src, entries=None):
        return list(dst), list(src), entries

    def copy(pool, dst, src, entries=None):
        assert not {d.data_ptr() for d in dst} & {s.data_ptr() for s in src}
        assert len({d.data_ptr() for d in dst}) == len(dst)
        for i, (d, s) in enumerate(zip(dst, src)):
            e = d.size(3) if entries is None else entries[i]
            d[:, :, :, :e] = s[:, :, :, :e]

    monkeypatch.setattr(kvcache, "_page_tables", tables)
    monkeypatch.setattr(kvcache, "copy_pages", copy)


def _tokens(c):
    return [int(p[0, 0, 0, e, 0]) for i, p in enumerate(c.pages) for e in range(min(c.pool.page_len, c.seqlen - 4 * i))]


def _write(c, n, value):
    for pos in range(c.seqlen - n, c.seqlen):
        c.pages[pos // 4][0, 0, 0, pos % 4, 0] = value


def test_holders_of_a_page():
    pool = _pool()
    p = pool.alloc_page()
    assert pool.page_holders(p) == 1
    pool.share_page(p)
    assert pool.page_holders(p) == 2 and pool.num_pages == 1
    pool.free_page(p)
    pool.free_page(p)
    assert pool.page_holders(p) == 0 and pool.num_pages == 0
    with pytest.raises(KeyError):
        pool.free_page(p)
    with pytest.raises(RuntimeError, match="not allocated"):
        pool.share_page(p)


def test_extend_and_acquire_agree():
    from loquetier_b200 import kvcache
    pool = _pool()
    a, b = kvcache.KvCache(pool, 3), kvcache.KvCache(pool, 3)
    for n in (0, 1, 1, 5, 9):
        a.extend(n)
        for _ in range(n):
            b.acquire_one()
        assert a.seqlen == b.seqlen and a.num_pages == b.num_pages
        assert a.ptrs.tolist() == [p.data_ptr() for p in a.pages]
    with pytest.raises(ValueError):
        a.extend(-1)
    for bad in (-1, a.seqlen + 1):
        with pytest.raises(ValueError):
            a.truncate(bad)


def test_random_lives_of_forked_caches(cpu_copies):
    """Random growth, forks, cuts, releases and compactions against lists of tokens: no cache ever sees another's tokens,
    every page is free or held as often as caches hold it."""
    from loquetier_b200 import kvcache
    for seed in range(30):
        r = random.Random(seed)
        pool = _pool(per_slab=r.choice([1, 3, 5]))
        live = [(kvcache.KvCache(pool, 0), [])]
        stamp = 0
        for _ in range(60):
            i = r.randrange(len(live))
            c, want = live[i]
            what = r.random()
            if what < 0.45:
                n, stamp = r.randint(0, 9), stamp + 1
                c.extend(n)
                _write(c, n, stamp)
                live[i] = (c, want + [stamp] * n)
            elif what < 0.6:
                n = r.randint(0, c.seqlen)
                c.truncate(n)
                live[i] = (c, want[:n])
            elif what < 0.75 and len(live) < 12:
                live += [(k, list(want)) for k in c.fork(r.randint(0, 3))]
            elif what < 0.85:
                some = [x for x, _ in live if r.random() < 0.8]
                slabs = pool.num_slabs
                assert pool.compact(some) == slabs - pool.num_slabs
            elif len(live) > 1:
                c.release()
                del live[i]
            held = {}
            for x, tokens in live:
                assert x.seqlen == len(tokens) and _tokens(x) == tokens
                assert x.ptrs.tolist() == [p.data_ptr() for p in x.pages]
                for p in x.pages:
                    held[p.data_ptr()] = held.get(p.data_ptr(), 0) + 1
            assert pool.num_pages == len(held) and all(pool.page_holders(p) == held[p.data_ptr()]
                                                       for p in pool.allocated_pages())
            assert len(pool._free) + pool.num_pages == pool.num_slabs * pool._pages_per_slab
        if pool.num_slabs:
            pool.compact([c for c, _ in live])
            assert pool.num_slabs == -(-pool.num_pages // pool._pages_per_slab)


def test_a_fork_that_fails_gives_its_pages_back(cpu_copies, monkeypatch):
    from loquetier_b200 import kvcache
    pool = _pool()
    c = kvcache.KvCache(pool, 6)

    def broken(*a):
        raise RuntimeError("no")

    monkeypatch.setattr(kvcache, "copy_pages", broken)
    with pytest.raises(RuntimeError, match="no"):
        c.fork(3)
    assert pool.num_pages == 2 and pool.page_holders(c.pages[0]) == 1


def test_caches_of_another_pool_are_refused():
    from loquetier_b200 import kvcache
    a, b = _pool(), _pool()
    ca, cb = kvcache.KvCache(a, 4), kvcache.KvCache(b, 4)
    with pytest.raises(RuntimeError, match="same pool"):
        kvcache.fork_caches([ca, cb])
    with pytest.raises(RuntimeError, match="of this pool"):
        a.compact([cb])
    with pytest.raises(ValueError):
        ca.fork(-1)
    assert kvcache.fork_caches([]) == [] and ca.fork(0) == []
    assert [k.seqlen for k in ca.fork(2)] == [4, 4]        # a full page: nothing to copy


def test_c_abi_refusals():
    """Checked on the host before any CUDA call."""
    from loquetier_b200 import cabi
    L = cabi.lib
    ws = L.smlm_b200_batch_extend_workspace_bytes(2, 8, 64, 16, 32, 8)
    assert ws > 0 and L.smlm_b200_batch_extend_workspace_bytes(0, 8, 64, 16, 32, 8) == 0
    assert L.smlm_b200_batch_extend_workspace_bytes(1, 4, 2, 16, 300, 300) == 0     # a CTA per kv head: nothing is cut

    def ext(o=512, wsp=256, bytes_=ws, rows=8, pages=64, nq=32, hd=128, layer=0, P=16, theta=10000.0, dt=1, batch=2):
        return L.smlm_b200_batch_extend(o, 256, 256, 256, 256, 256, wsp, bytes_, None, batch, rows, pages, nq, 8, hd, 1, layer,
                                        P, theta, dt, None)

    assert ext(dt=7) == 2 and ext(hd=64) == 3 and ext(P=128) == 3 and ext(P=12) == 3 and ext(nq=40) == 3 and ext(nq=36) == 3
    assert ext(layer=1) == 1 and ext(theta=0.0) == 1 and ext(rows=-1) == 1 and ext(o=None) == 1
    assert ext(o=264) == 4 and ext(wsp=264) == 4
    assert ext(o=256) == 1   # in place
    assert ext(wsp=None) == 5 and ext(bytes_=ws - 1) == 5
    assert ext(rows=1 << 28) == 1 and ext(pages=1 << 28) == 1
    assert ext(batch=0) == 0 and ext(rows=0) == 0

    def cp(dst=256, n=3, hd=128, P=16, dt=0, layers=2):
        return L.smlm_b200_copy_pages(dst, 256, None, None, n, layers, 8, hd, P, dt, None)

    assert cp(dst=None) == 1 and cp(n=-1) == 1 and cp(layers=0) == 1 and cp(hd=64) == 3 and cp(P=128) == 3 and cp(dt=4) == 2
    assert cp(n=0) == 0 and cp(layers=1 << 20) == 1

    def fwd(yq=256, q=256, wq=256, wk=256, pos=256, qs=4096, ks=1024, T=4, hd=128, theta=1e4, dt=1):
        return L.smlm_b200_qk_norm_rope(yq, 256, q, 256, wq, wk, pos, qs, ks, T, 32, 8, hd, 0, theta, 1e-6, dt, None)

    assert fwd(yq=None) == 1 and fwd(q=None) == 1 and fwd(wq=None) == 1 and fwd(theta=0.0) == 1 and fwd(T=-1) == 1
    assert fwd(wq=None, wk=None, pos=None) == 1 and fwd(qs=4088) == 1 and fwd(ks=1000) == 1
    assert fwd(q=264) == 4 and fwd(yq=264) == 4 and fwd(wk=264) == 4 and fwd(qs=4100) == 4
    assert fwd(hd=64) == 3 and fwd(dt=9) == 2 and fwd(T=0) == 0
    need = L.smlm_b200_qk_norm_rope_bwd_workspace_bytes(4, 32, 8)
    assert need > 0 and L.smlm_b200_qk_norm_rope_bwd_workspace_bytes(0, 32, 8) == 0

    def bwd(dq=256, dwq=256, gq=256, wsp=256, bytes_=need, T=4):
        return L.smlm_b200_qk_norm_rope_bwd(dq, 256, dwq, 256, gq, 256, 256, 256, 256, 256, 256, wsp, bytes_, 4096, 1024, T,
                                            32, 8, 128, 0, 1e4, 1e-6, 1, None)

    assert bwd(dq=None) == 1 and bwd(dwq=None) == 1 and bwd(T=0) == 1 and bwd(gq=264) == 4
    assert bwd(dwq=None, wsp=None) == 1   # one gradient of the two
    assert bwd(wsp=None) == 5 and bwd(bytes_=need - 1) == 5 and bwd(wsp=264) == 4

    def app(yq=256, v=256, wq=256, vs=1024, ind=256, batch=2, T=5, P=16, layer=0):
        return L.smlm_b200_norm_append_kv(yq, 256, 256, v, wq, 256, 256, 256, 256, ind, None, 4096, 1024, vs, batch, T, 9, 32,
                                          8, 128, 1, layer, P, 1e-6, 1, None)

    assert app(yq=None) == 1 and app(v=None) == 1 and app(wq=None) == 1 and app(vs=1000) == 1 and app(layer=1) == 1
    assert app(ind=None) == 1                     # one token per request, but five tokens for two
    assert app(yq=264) == 4 and app(v=264) == 4 and app(vs=1028) == 4 and app(P=24) == 3
    assert app(T=0) == 0 and app(batch=0) == 0


def test_wrappers_refuse_before_they_launch():
    from loquetier_b200 import kvcache
    from loquetier_b200.kernel_utils import qk_norm_rope
    pool = _pool()
    kv = kvcache.BatchedKvCache([kvcache.KvCache(pool, 5)])
    q = torch.zeros((1, 2, 128))
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        kvcache.batch_extend(q, torch.tensor([0, 1], dtype=torch.int32), kv, 1e4, 0)
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        kvcache.norm_append_kv(kv, q, q, q, q[0, 0], q[0, 0], 1e-6, 0)
    with pytest.raises(RuntimeError, match="dst must be a CUDA tensor"):
        kvcache.copy_pages(pool, torch.zeros(1, dtype=torch.int64), torch.zeros(1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        qk_norm_rope.apply(q, q, None, None, torch.zeros(1, dtype=torch.int32))


def test_gradient_formulas_against_differences():
    """The formulas that the kernels are compared with are the derivatives of the definition: central differences in
    float64, h = 1e-6, good to h^2 and 2^-52 / h."""
    g = torch.Generator().manual_seed(1)
    x, w, dy = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((3, 2, 128), (128,), (3, 2, 128)))
    pos = torch.tensor([0, 5, 9001])
    for weight in (w, None):
        for at in (pos, None):
            if weight is None and at is None:
                continue
            dx, dw, _ = R.norm_rope_grads(x, weight, at, dy, 1e4, 1e-6)
            f = lambda x_, w_: (R.norm_rope(x_, w_, at, 1e4, 1e-6) * dy).sum()
            h = 1e-6
            for idx in ((0, 0, 0), (1, 1, 70), (2, 0, 127), (2, 1, 64)):
                e = torch.zeros_like(x)
                e[idx] = h
                assert abs((f(x + e, weight) - f(x - e, weight)) / (2 * h) - dx[idx]) < 1e-6
            if weight is not None:
                for i in (0, 63, 64, 127):
                    e = torch.zeros_like(w)
                    e[i] = h
                    assert abs((f(x, w + e) - f(x, w - e)) / (2 * h) - dw[i]) < 1e-6
