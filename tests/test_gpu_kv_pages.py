"""Page copies and what is built on them - forks, truncation, compaction - and a run of the operators around a shared cache
as a server would make it.  Copies are bit-exact."""
import pytest
import torch

import shared_cache_ref as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BASE, EPS = 10000.0, 1e-6


def _pool(layers=2, heads=3, P=16, dtype=torch.bfloat16, per_slab=8):
    from loquetier_b200 import kvcache
    return kvcache.KvPool(layers, heads, 128, P, dtype, DEV, pages_per_slab=per_slab)


def _fill(pages, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    for p in pages:
        p.copy_(torch.randn(p.shape, generator=g, device=DEV))


def _ptrs(pages):
    return torch.tensor([p.data_ptr() for p in pages], dtype=torch.int64, device=DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layers,heads,P", [(1, 1, 8), (2, 3, 16), (32, 8, 16), (5, 2, 64), (3, 7, 32)])
@pytest.mark.parametrize("whole", [True, False])
def test_copy_pages(dtype, layers, heads, P, whole):
    from loquetier_b200 import kvcache
    pool = _pool(layers, heads, P, dtype, per_slab=5)
    src = [pool.alloc_page() for _ in range(3)]
    dst = [pool.alloc_page() for _ in range(8)]
    _fill(src + dst, 1)
    before = [d.clone() for d in dst]
    pick = [0, 1, 1, 2, 0, 2, 1, 0]
    entries = [P, 1, P - 1, 0, P // 2, 3, 5, P]
    kept = [s.clone() for s in src]
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    kvcache.copy_pages(pool, _ptrs(dst), _ptrs([src[i] for i in pick]),
                       None if whole else torch.tensor(entries, dtype=torch.int32, device=DEV), status_word=word)
    torch.cuda.synchronize()
    assert int(word.item()) == 0
    for d, b, i, e in zip(dst, before, pick, entries):
        e = P if whole else e
        assert torch.equal(d[..., :e, :], kept[i][..., :e, :]) and torch.equal(d[..., e:, :], b[..., e:, :])
    assert all(torch.equal(s, t) for s, t in zip(src, kept))


def test_copy_of_many_pages_and_of_none():
    from loquetier_b200 import kvcache
    pool = _pool(1, 1, 8, per_slab=4096)
    src, dst = ([pool.alloc_page() for _ in range(70000)] for _ in range(2))
    slab = pool._slabs[0]
    for i, s in enumerate(pool._slabs):
        s.copy_(torch.randint(-1000, 1000, s.shape, device=DEV) + i)
    a, b = _ptrs(src), _ptrs(dst)
    kvcache.copy_pages(pool, b, a)
    kvcache.copy_pages(pool, b[:0], a[:0])
    torch.cuda.synchronize()
    for i in (0, 1, 65534, 65535, 65536, 69999):
        assert torch.equal(src[i], dst[i])


def test_copy_reports_bad_entries_and_skips_them():
    from loquetier_b200 import kvcache
    pool = _pool()
    pages = [pool.alloc_page() for _ in range(6)]
    _fill(pages, 2)
    before = [p.clone() for p in pages]
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    dst, src = _ptrs(pages[3:]), _ptrs(pages[:3])
    dst[0] = 0
    kvcache.copy_pages(pool, dst, src, torch.tensor([4, 17, 16], dtype=torch.int32, device=DEV), status_word=word)
    torch.cuda.synchronize()
    assert int(word.item()) == 3
    assert torch.equal(pages[3], before[3]) and torch.equal(pages[4], before[4]) and torch.equal(pages[5], before[2])
    word.zero_()
    src[1] += 4
    kvcache.copy_pages(pool, _ptrs(pages[3:]), src, torch.tensor([0, 16, -1], dtype=torch.int32, device=DEV), status_word=word)
    torch.cuda.synchronize()
    assert int(word.item()) == 3
    assert torch.equal(pages[3], before[3]) and torch.equal(pages[4], before[4]) and torch.equal(pages[5], before[2])


def _dense(cache, layer):
    if not cache.pages:
        return torch.empty((2, 0, cache.pool.num_heads, 128), device=DEV)
    return torch.cat([p[layer] for p in cache.pages], dim=2)[:, :, :cache.seqlen].transpose(1, 2)


def _tables_match(cache):
    assert cache.ptrs.tolist() == [p.data_ptr() for p in cache.pages]


@pytest.mark.parametrize("length", [0, 1, 15, 16, 17, 32, 50])
def test_forks_hold_the_same_tokens_and_part_ways(length):
    from loquetier_b200 import kvcache
    pool = _pool(per_slab=4)
    c = kvcache.KvCache(pool, length)
    _fill(c.pages, length + 1)
    want = _dense(c, 1).clone()
    kids = c.fork(3)
    assert pool.num_pages == c.num_pages + (3 if length % 16 else 0)
    for kid in kids:
        assert kid.seqlen == length and torch.equal(_dense(kid, 1), want)
        _tables_match(kid)
    # each goes its own way: new tokens of one are not seen by the others
    g = torch.Generator(device=DEV).manual_seed(9)
    tails = []
    for kid in [c] + kids:
        kid.extend(20)
        kv = kvcache.BatchedKvCache([kid])
        k, v = (torch.randn((20, 3, 128), generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
        kvcache.init_kv(kv, k, v, torch.tensor([0, 20], dtype=torch.int32, device=DEV), 1)
        tails.append(torch.stack([k, v]))
    torch.cuda.synchronize()
    for kid, tail in zip([c] + kids, tails):
        assert torch.equal(_dense(kid, 1), torch.cat([want, tail], dim=1))
        _tables_match(kid)
    c.release()
    for kid in kids[1:]:
        kid.release()
    assert torch.equal(_dense(kids[0], 1), torch.cat([want, tails[1]], dim=1))
    kids[0].release()
    assert pool.num_pages == 0


def test_truncation_into_a_shared_page_leaves_the_others_alone():
    from loquetier_b200 import kvcache
    pool = _pool()
    c = kvcache.KvCache(pool, 40)
    _fill(c.pages, 3)
    want = _dense(c, 0).clone()
    kid, = c.fork()
    kid.truncate(21)                     # into the second page, which both hold
    assert kid.seqlen == 21 and kid.num_pages == 2 and torch.equal(_dense(kid, 0), want[:, :21])
    _tables_match(kid)
    kid.extend(3)
    kv = kvcache.BatchedKvCache([kid])
    one = torch.ones((3, 3, 128), dtype=torch.bfloat16, device=DEV)
    kvcache.init_kv(kv, one, one, torch.tensor([0, 3], dtype=torch.int32, device=DEV), 0)
    assert torch.equal(_dense(c, 0), want) and (_dense(kid, 0)[:, 21:] == 1).all()
    kid.truncate(16)                     # to a full page: nothing to copy, still shared
    assert kid.pages[0].data_ptr() == c.pages[0].data_ptr() and pool.page_holders(c.pages[0]) == 2
    kid.truncate(0)
    assert kid.num_pages == 0 and pool.num_pages == 3 and torch.equal(_dense(c, 0), want)


def test_compaction_moves_pages_and_keeps_the_tokens():
    from loquetier_b200 import kvcache
    pool = _pool(per_slab=4)
    caches = [kvcache.KvCache(pool, 40) for _ in range(8)]          # 24 pages in 6 slabs
    for i, c in enumerate(caches):
        _fill(c.pages, i)
    kid, = caches[5].fork()
    for i in (0, 2, 3, 6):
        caches[i].release()
    live = [caches[i] for i in (1, 4, 5, 7)] + [kid]
    want = [_dense(c, 1).clone() for c in live]
    before = pool.num_slabs
    assert pool.compact(live[:-1]) < before          # the fork's pages are held by a cache that is not named: they stay
    assert all(torch.equal(_dense(c, 1), w) for c, w in zip(live, want))
    given = pool.compact(live)
    torch.cuda.synchronize()
    assert pool.num_slabs == -(-pool.num_pages // 4) and given + pool.num_slabs <= before
    for c, w in zip(live, want):
        assert torch.equal(_dense(c, 1), w)
        _tables_match(c)
    assert pool.compact(live) == 0
    more = kvcache.KvCache(pool, 100)
    assert len({p.data_ptr() for c in live + [more] for p in c.pages}) == pool.num_pages
    for c in live + [more]:
        c.release()
    assert pool.num_pages == 0
    pool.compact([])
    assert pool.num_slabs == 0


def test_copies_under_capture_are_refused():
    from loquetier_b200 import kvcache
    pool = _pool()
    c = kvcache.KvCache(pool, 20)
    kid, = c.fork()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (c.fork, lambda: c.truncate(5), lambda: pool.compact([c, kid])):
            with pytest.raises(RuntimeError, match="cannot be captured"):
                call()
    assert c.seqlen == 20 and pool.num_pages == 3


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_served_step_from_prompt_to_verified_drafts(dtype):
    """A prompt is normalised into the cache and attended to, continued three ways with drafts of different lengths, the
    drafts are verified, some rejected, the pool is drawn together, and the next tokens follow - every attention result
    against the definition on the tokens each continuation really has."""
    from loquetier_b200 import kvcache
    N, G, P, layer = 2, 4, 16, 1
    pool = kvcache.KvPool(2, N, 128, P, dtype, DEV, pages_per_slab=2)
    g = torch.Generator(device=DEV).manual_seed(5)
    wq, wk = ((1 + 0.3 * torch.randn(128, generator=g, device=DEV)).to(dtype) for _ in range(2))

    def step(caches, new):
        """New tokens of every cache: into the pages and attended from.  Returns what the cache now holds, per cache."""
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        for c, n in zip(caches, new):
            c.extend(n)
        kv = kvcache.BatchedKvCache(caches)
        ind = torch.tensor(starts, dtype=torch.int32, device=DEV)
        qkv = torch.randn((starts[-1], N * G + 2 * N, 128), generator=g, device=DEV).to(dtype)
        q, k, v = qkv[:, :N * G], qkv[:, N * G:N * G + N], qkv[:, N * G + N:]
        nq = kvcache.norm_append_kv(kv, q, k, v, wq, wk, EPS, layer, ind)
        o = kvcache.batch_extend(nq, ind, kv, BASE, layer)
        nk = R.head_norm(k, wk, EPS)
        for i, c in enumerate(caches):
            held = _dense(c, layer)
            bound = R.norm_rope_bound(k[starts[i]:starts[i + 1]], wk, None, BASE, EPS, dtype)
            assert ((held[0, c.seqlen - new[i]:].double() - nk[starts[i]:starts[i + 1]]).abs() <= bound).all()
            assert torch.equal(held[1, c.seqlen - new[i]:], v[starts[i]:starts[i + 1]])
        want, bound = R.extend(nq, starts, [tuple(_dense(c, layer)) for c in caches], BASE)
        R.check_extend(o, want, bound, dtype, f"step {new}")

    spare = kvcache.KvCache(pool, 100)
    prompt = kvcache.KvCache(pool, 0)
    step([prompt], [150])
    spare.release()
    history = _dense(prompt, layer).clone()
    kids = prompt.fork(3)
    step(kids, [4, 1, 9])
    kids[0].truncate(151)
    kids[2].truncate(154)
    assert pool.compact([prompt] + kids) > 0
    step(kids, [3, 20, 1])
    kids[1].truncate(140)                       # back into the shared prompt
    step(kids, [1, 1, 1])
    assert torch.equal(_dense(prompt, layer), history)
    for c in [prompt] + kids:
        c.release()
    assert pool.num_pages == 0
