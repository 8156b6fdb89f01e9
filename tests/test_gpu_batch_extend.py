"""Attention of a chunk of new tokens over the paged cache (``kvcache.batch_extend``) against its definition in 64 bits.
Tolerances: ``shared_cache_ref.extend`` (elementwise, by arithmetic) and ``check_extend`` (as a whole)."""
import random

import pytest
import torch

import shared_cache_ref as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BASE = 10000.0
LAYERS, LAYER = 2, 1


def _batch(seed, lens, new, N, G, P, dtype, poison=True, scale=1.0):
    """Caches of ``lens`` keys on shuffled pages; unused entries and the other layer hold NaN.  Returns what the operator
    takes and the caches' dense keys and values."""
    from loquetier_b200 import kvcache
    g = torch.Generator(device=DEV).manual_seed(seed)
    npages = [-(-L // P) for L in lens]
    total = sum(npages)
    pool = torch.full((max(total, 1), LAYERS, 2, N, P, 128), float("nan") if poison else 0.0, dtype=dtype, device=DEV)
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    table, dense, at = [], [], 0
    for L, n in zip(lens, npages):
        ids = order[at:at + n]
        at += n
        K = (torch.randn((L, N, 128), generator=g, device=DEV) * scale).to(dtype)
        V = torch.randn((L, N, 128), generator=g, device=DEV).to(dtype)
        for j, i in enumerate(ids):
            m = min(P, L - j * P)
            pool[i, LAYER, 0, :, :m] = K[j * P:j * P + m].transpose(0, 1)
            pool[i, LAYER, 1, :, :m] = V[j * P:j * P + m].transpose(0, 1)
        table += ids
        dense.append((K, V))
    starts, ind = [0], [0]
    for n, p in zip(new, npages):
        starts.append(starts[-1] + n)
        ind.append(ind[-1] + p)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    q = torch.randn((starts[-1] + 2, N * G, 128), generator=g, device=DEV).to(dtype)   # two rows of no request behind
    args = dict(q=q, qo_indptr=i32(starts), kv_ptrs=torch.tensor([pool[i].data_ptr() for i in table], dtype=torch.int64,
                                                                 device=DEV),
                kv_indptr=i32(ind), last_page_offset=i32([(L - 1) % P + 1 if L else 0 for L in lens]), num_layers=LAYERS,
                layer_idx=LAYER, num_kv_heads=N, base=BASE, page_size=P)
    return pool, args, starts, dense


def _run(args, expect=0, **kw):
    from loquetier_b200 import kvcache
    o = torch.full(args["q"].shape, 7.0, dtype=args["q"].dtype, device=DEV)
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    kvcache.batch_extend_into(o, status_word=word, **{**args, **kw})
    torch.cuda.synchronize()
    assert int(word.item()) == expect, f"fault bits {int(word.item())}"
    return o


def _check(seed, lens, new, N, G, P, dtype, scale=1.0):
    pool, args, starts, dense = _batch(seed, lens, new, N, G, P, dtype, scale=scale)
    o = _run(args)
    want, bound = R.extend(args["q"], starts, dense, BASE)
    R.check_extend(o, want, bound, dtype, f"{lens} {new}")
    assert (o[starts[-1]:] == 7.0).all()          # rows of no request are left as they were
    assert torch.equal(o, _run(args))             # the same bits again
    return pool, args, starts, o


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group,page", [(1, 16), (2, 8), (4, 16), (8, 64), (4, 32), (1, 8)])
@pytest.mark.parametrize("most", [1, 3, 8, 40])
def test_ragged_chunks(dtype, group, page, most):
    """Chunks of nothing, of one token and of the whole cache beside longer ones; caches that end inside a tile and a
    page, and one without a key."""
    r = random.Random(100 * group + page + most)
    new = [r.randint(1, most) for _ in range(5)] + [0, most, 1, 0]
    lens = [n + r.choice([0, 1, 15, 16, 17, 63, 64, 65, 200]) for n in new[:5]] + [33, most, 1, 0]
    _check(most, lens, new, 2, group, page, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [(8, 4), (1, 8), (3, 1)])
@pytest.mark.parametrize("new,length", [(1, 5003), (2, 5003), (7, 9001), (17, 4099), (33, 2500), (130, 3333)])
def test_one_long_cache_is_cut_into_ranges(dtype, heads, new, length):
    _check(new, [length], [new], *heads, 16, dtype)


@pytest.mark.parametrize("rows", [1, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257])
def test_rows_at_the_edges_of_tiles(rows):
    """One kv head, one query head: as many rows as new tokens."""
    _check(rows, [rows + 50, rows, 700 + rows], [rows, rows, rows], 1, 1, 16, torch.bfloat16)


def test_far_positions_lose_nothing():
    """A cache of 70 000 keys: single-precision angles would be off by hundredths of a radian there."""
    _check(5, [70001], [3], 1, 4, 64, torch.float16)


@pytest.mark.parametrize("requests,most,heads", [(300, 4, (2, 4)), (700, 3, (1, 8)), (3000, 2, (1, 1)), (700, 12, (1, 4)),
                                                  (400, 30, (2, 4)), (300, 90, (1, 8))])
def test_uneven_batch_of_many_requests(requests, most, heads):
    """More requests than a CTA looks at together and more row tiles in a share than are laid out at a time; many without
    a new token, one far longer than the rest."""
    r = random.Random(requests)
    new = [r.choice([0, r.randint(0, most), most]) for _ in range(requests)]
    lens = [n + r.randint(0, 90) for n in new]
    lens[217] = 6000
    _check(requests, lens, new, *heads, 16, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,page", [((2, 4), 16), ((1, 8), 8), ((3, 2), 64), ((4, 1), 32)])
def test_long_chunks_whose_keys_are_rotated_in_front(dtype, heads, page):
    """Several row tiles per request: whole prompts, pieces of prompts, beside an empty request and one of a token."""
    n = 1300 // heads[1]
    _check(page, [n, n + 777, 0, 3 * n + 5, 64, n + 1], [n, n, 0, n + 3, 1, n], *heads, page, dtype)


def test_large_scores():
    """Keys twenty times larger: a softmax that is all but one key, maxima that keep rising."""
    pool, args, starts, dense = _batch(7, [900, 77], [5, 9], 2, 4, 16, torch.float16, scale=20.0)
    o = _run(args)
    want, bound = R.extend(args["q"], starts, dense, BASE)
    rows = slice(0, starts[-1])
    assert ((o.double()[rows] - want[rows]).abs() <= bound[rows]).all()


def test_a_longer_page_table_changes_nothing():
    pool, args, starts, o = _check(8, [300, 2000, 17], [4, 6, 1], 2, 4, 16, torch.bfloat16)
    padded = torch.cat([args["kv_ptrs"], args["kv_ptrs"][:1].expand(500)]).contiguous()
    assert torch.equal(o, _run(args, kv_ptrs=padded))


@pytest.mark.parametrize("group", [1, 4, 8])
def test_agrees_with_decode_and_prefill(group):
    """One new token per request is the decode operator's case, whole prompts are the prefill operator's.  Each is within
    the whole-error bound of the definition (moderate positions), so they are within twice that of one another."""
    from loquetier_b200 import kvcache
    P, N, dt = 16, 2, torch.bfloat16
    for new in ([1, 1, 1], [40, 333, 17]):
        lens = [40, 333, 17]
        pool, args, starts, dense = _batch(10 + group, lens, new, N, group, P, dt, poison=False)
        args["q"] = args["q"][:starts[-1]].contiguous()
        o = _run(args).double()
        ref = torch.empty_like(args["q"])
        common = (args["kv_ptrs"], args["kv_indptr"], args["last_page_offset"], LAYERS, LAYER, N, BASE, P)
        if new[0] == 1:
            kvcache.batch_decode_into(ref, args["q"], *common)
        else:
            kvcache.batch_prefill_into(ref, args["q"], args["qo_indptr"], *common)
        assert ((o - ref.double()).norm() / o.norm()).item() <= 2.6 * R.unit(dt)


def test_captured_graph_follows_new_lengths():
    """A captured call replays with other lengths, queries and pages, beside a second graph of its own."""
    N, G, P, dt = 2, 4, 16, torch.bfloat16
    pool, args, starts, dense = _batch(21, [500, 64, 2000], [3, 5, 2], N, G, P, dt)
    pool2, args2, starts2, dense2 = _batch(22, [100, 1700, 90], [5, 2, 3], N, G, P, dt)
    from loquetier_b200 import kvcache
    names = ("q", "qo_indptr", "kv_indptr", "last_page_offset")
    ptrs = torch.zeros(max(args["kv_ptrs"].numel(), args2["kv_ptrs"].numel()), dtype=torch.int64, device=DEV)
    graphs = []
    for first in (args, args2):
        held = {**first, **{n: first[n].clone() for n in names}, "kv_ptrs": ptrs.clone()}
        held["kv_ptrs"][:first["kv_ptrs"].numel()] = first["kv_ptrs"]
        o = torch.full(held["q"].shape, 7.0, dtype=dt, device=DEV)
        kvcache.batch_extend_into(o, **held)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kvcache.batch_extend_into(o, **held)
        graphs.append((graph, held, o))
    for turn in range(2):
        for (graph, held, o), now in zip(graphs, (args, args2) if turn == 0 else (args2, args)):
            for n in names:
                held[n].copy_(now[n])
            held["kv_ptrs"][:now["kv_ptrs"].numel()].copy_(now["kv_ptrs"])
            o.fill_(7.0)
            graph.replay()
        torch.cuda.synchronize()
        for (graph, held, o), now in zip(graphs, (args, args2) if turn == 0 else (args2, args)):
            want, bound = R.extend(now["q"], (starts, starts2)[now is args2], (dense, dense2)[now is args2], BASE)
            R.check_extend(o, want, bound, dt, "replayed")


def test_two_streams_at_once():
    """Calls on two streams share nothing: results equal those one after the other."""
    pools = [_batch(30 + i, [3000 - 500 * i, 40], [5, 3], 2, 4, 16, torch.bfloat16) for i in range(2)]
    work = [p[1] for p in pools]
    alone = [_run(a) for a in work]
    from loquetier_b200 import kvcache
    outs = [[torch.full(a["q"].shape, 7.0, dtype=a["q"].dtype, device=DEV) for _ in range(20)] for a in work]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for i in range(20):
        for s, a, o in zip(streams, work, outs):
            with torch.cuda.stream(s):
                kvcache.batch_extend_into(o[i], **a)
    torch.cuda.synchronize()
    for want, got in zip(alone, outs):
        assert all(torch.equal(want, o) for o in got)


def test_bad_tables_are_reported_not_followed():
    pool, args, starts, dense = _batch(40, [20, 20], [3, 2], 2, 4, 16, torch.bfloat16)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    want, bound = R.extend(args["q"], starts, dense, BASE)
    for kw, expect in ((dict(kv_indptr=i32([0, 2, 9])), 1), (dict(kv_indptr=i32([0, -3, 4])), 1),
                       (dict(qo_indptr=i32([0, 3, 900])), 1), (dict(qo_indptr=i32([-1, 3, 5])), 1),
                       (dict(last_page_offset=i32([4, 17])), 1)):
        _run(args, expect=expect, **kw)
    ptrs = args["kv_ptrs"].clone()
    ptrs[1] = 0
    _run(args, expect=2, kv_ptrs=ptrs)
    ptrs[1] = args["kv_ptrs"][1] + 8
    o = _run(args, expect=2, kv_ptrs=ptrs)
    R.check_extend(o[3:5], want[3:5], bound[3:5], torch.bfloat16, "the sound request beside a bad one")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,length,group,far", [(5, 300, 4, 1), (40, 300, 1, 7), (70, 2000, 8, 30), (200, 200, 4, 100), (3, 9000, 8, 2)])
def test_what_is_not_finite_reaches_only_those_who_see_it(dtype, new, length, group, far):
    """NaN and infinities among the new tokens' keys and values: earlier tokens are as if they were not there."""
    pool, args, starts, dense = _batch(50 + new, [length, 77], [new, 3], 2, group, 16, dtype)
    clean = _run(args)
    at = length - far                                   # the token whose value is spoilt, seen from query new - far on
    def spoil(which, position, head, dims, value):
        page = args["kv_ptrs"].tolist().index(args["kv_ptrs"][position // 16].item())
        ids = [i for i in range(pool.size(0)) if pool[i].data_ptr() == args["kv_ptrs"][page].item()]
        pool[ids[0], LAYER, which, head, position % 16, dims] = value
    spoil(1, at, 0, slice(3, 5), float("nan"))
    spoil(1, at, 1, slice(127, 128), float("-inf"))
    if far > 1:
        spoil(1, length - 1, 1, slice(0, 1), float("inf"))
        spoil(0, length - 1, 0, slice(9, 10), float("nan"))
    o = _run(args)
    first = new - far
    assert torch.equal(o[:first], clean[:first]) and torch.equal(o[new:], clean[new:])
    seen, G = o[first:new], group
    assert torch.isnan(seen[:, :G, 3:5]).all() and (seen[:, G:, 127] == float("-inf")).all()
    last = new - 1
    keep = torch.ones(128, dtype=torch.bool, device=DEV)
    keep[3:5] = False
    rows = slice(first, last if far > 1 else new)
    assert torch.equal(o[rows, :G][..., keep], clean[rows, :G][..., keep])
    assert torch.equal(o[rows, G:, :127], clean[rows, G:, :127])
    if far > 1:
        assert torch.isnan(o[last, :G]).all() and (o[last, G:, 0] == float("inf")).all()
        assert torch.equal(o[last, G:, 1:127], clean[last, G:, 1:127])


def test_more_queries_than_keys():
    """Rows that see no key are zeros, the others as the definition has them; the status word tells."""
    pool, args, starts, dense = _batch(41, [3, 30], [3, 4], 2, 4, 16, torch.float16)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    o = _run(args, expect=1, last_page_offset=i32([1, 14]))
    assert (o[:2] == 0).all()                                   # positions -2 and -1
    assert torch.equal(o[2].float(), dense[0][1][0].repeat_interleave(4, 0).float())   # sees one key: its value
    full, bd = R.extend(args["q"], starts, dense, BASE)
    R.check_extend(o[3:7], full[3:7], bd[3:7], torch.float16, "the request beside it")


def test_an_empty_batch_of_pages_gives_zeros():
    from loquetier_b200 import kvcache
    q = torch.randn((2, 8, 128), device=DEV).to(torch.bfloat16)
    o = torch.full_like(q, 7.0)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    kvcache.batch_extend_into(o, q, i32([0, 2]), torch.empty(0, dtype=torch.int64, device=DEV), i32([0, 0]), i32([0]), 1, 0, 2,
                              BASE, 16, status_word=word)
    torch.cuda.synchronize()
    assert int(word.item()) == 1 and (o == 0).all()
