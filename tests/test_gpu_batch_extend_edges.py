"""``kvcache.batch_extend`` at the edges of its range."""
import math
import random

import pytest
import torch

import shared_cache_ref as R
from extend_whole import check_whole
from test_gpu_batch_extend import BASE, DEV, LAYER, _batch, _check, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,length,group", [(1, 1, 1), (3, 40, 4), (5, 5000, 4), (70, 300, 2), (150, 2000, 4)])
def test_scores_that_leave_the_range(new, length, group):
    """Where every score that a row sees is -inf the definition has no answer, and NaN says so; a row that sees one key with
    a finite score has that key's value.  Only the slowest pair of dimensions is set (over 5000 keys it turns by 0.6), to 1e20:
    all products are about -1e40 / sqrt(128)."""
    pool, args, starts, dense = _batch(new, [length], [new], 1, group, 16, torch.bfloat16)
    args["q"].zero_()
    args["q"][..., 63] = 1e20
    pool[:, LAYER, 0] = 0
    pool[:, LAYER, 0, :, :, 63] = -1e20
    o = _run(args)
    assert torch.isnan(o[:new]).all() and (o[new:] == 7.0).all()
    at = length // 2                                     # this key scores zero
    where = [i for i in range(pool.size(0)) if pool[i].data_ptr() == args["kv_ptrs"][at // 16].item()][0]
    pool[where, LAYER, 0, :, at % 16] = 0
    o = _run(args)
    first = max(0, at - (length - new))                  # the first query that sees it
    assert torch.isnan(o[:first]).all()
    assert torch.equal(o[first:new], dense[0][1][at].expand_as(o[first:new]))


@pytest.mark.parametrize("requests,new,heads", [(20, 3, (296, 1)), (32, 5, (200, 4)), (31, 100, (64, 1)), (7, 700, (40, 1)),
                                                (32, 300, (74, 1))])
def test_few_requests_of_more_runs_than_are_laid_out_at_a_time(requests, new, heads):
    """Many kv heads leave each of them few CTAs, so that a share holds more row tiles than one round (16, or 4 of 64 rows and
    more).  Up to 32 requests are searched by one warp."""
    r = random.Random(requests)
    runs = [r.randint(max(1, new // 2), new) for _ in range(requests)]
    _check(requests, [n + r.randint(0, 40) for n in runs], runs, *heads, 16, torch.bfloat16)


def test_results_right_beside_the_queries():
    """Results in front of the queries and behind them, in one allocation, without a byte between them; one byte group
    less is refused."""
    pool, args, starts, dense = _batch(60, [300, 50], [5, 3], 2, 4, 16, torch.bfloat16)
    args["q"] = q = args["q"][:starts[-1]].contiguous()
    want = _run(args)
    n = q.numel()
    from loquetier_b200 import kvcache
    room = torch.zeros(3 * n, dtype=q.dtype, device=DEV)
    args["q"] = room[n:2 * n].view(q.shape)
    for first in (0, 2 * n):
        args["q"].copy_(q)
        o = kvcache.batch_extend_into(room[first:first + n].view(q.shape), **args)
        assert torch.equal(o, want) and torch.equal(args["q"], q)
    for first in (8, 2 * n - 8, n):
        with pytest.raises(RuntimeError):
            kvcache.batch_extend_into(room[first:first + n].view(q.shape), **args)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [(8, 4), (1, 8), (3, 1), (1, 1)])
@pytest.mark.parametrize("new,length", [(1, 5003), (2, 5003), (7, 9001), (1, 20011), (17, 4099), (33, 2500), (130, 3333)])
def test_long_caches_as_acheck_whole(dtype, heads, new, length):
    """Few rows over many keys: values so small that the elementwise bounds would let a zero pass."""
    pool, args, starts, dense = _batch(new, [length], [new], *heads, 16, dtype)
    want, _ = R.extend(args["q"], starts, dense, BASE)
    check_whole(_run(args)[:new], want[:new], dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 31])
def test_small_batches_as_acheck_whole(dtype, rows):
    lens, new = [rows + 350, 900, 700 + rows], [rows, 1, rows]
    pool, args, starts, dense = _batch(rows, lens, new, 1, 1, 16, dtype)
    want, _ = R.extend(args["q"], starts, dense, BASE)
    o = _run(args)
    for t0, t1 in zip(starts, starts[1:]):
        check_whole(o[t0:t1], want[t0:t1], dtype)


@pytest.mark.parametrize("new", [3, 300])
def test_near_the_last_position(new):
    """A cache that ends 37 keys short of 2^24, its last 4096 keys the ones that count, at scores of 20 and some that hang
    on the rotation: single-precision angles, off by half a radian there, give another result.  (One page of keys that score
    zero and have no value stands in for all the pages in front: the table may name a page more than once.)

    Every key is the rotation back of a vector u_j, every query that of t_i, so that the scores are t_i . u_j whatever the
    position.  Bound as in ``shared_cache_ref.extend``, with 2^-13 in a pair's turn for the angles (sines good to 2^-19, 63
    steps of a recurrence that adds them up)."""
    P, L, near, dtype = 64, (1 << 24) - 37, 4096, torch.float16
    assert L % P and near % P == 0
    u = R.unit(dtype)
    g = torch.Generator(device=DEV).manual_seed(new)
    fast = torch.zeros(128, dtype=torch.float64, device=DEV)
    fast[:8] = fast[64:72] = 1.0                           # the eight fastest pairs
    ahead = -(-L // P) - near // P                         # pages in front
    pos = torch.arange(ahead * P, L, device=DEV)
    rand = lambda *s: torch.randn(s, generator=g, device=DEV, dtype=torch.float64)
    t = fast * (1 + 0.3 * rand(new, 1, 128))
    key = fast * 14.0 * (1 + 0.2 * rand(pos.numel(), 1, 128))   # scores of 14 * 16 / sqrt(128) or so
    value = rand(pos.numel(), 1, 128).to(dtype)
    q = R.rotate(t, -pos[-new:], BASE).to(dtype)
    k = R.rotate(key, -pos, BASE).to(dtype)
    pool = torch.zeros((1 + near // P, 1, 2, 1, P, 128), dtype=dtype, device=DEV)
    pad = torch.zeros(near, 1, 128, dtype=dtype, device=DEV)
    for i, x in enumerate((k, value)):
        pad[:pos.numel()] = x
        pool[1:, 0, i, 0] = pad.view(-1, P, 128)
    table = [0] * ahead + list(range(1, 1 + near // P))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    ptrs = pool.data_ptr() + torch.tensor(table, dtype=torch.int64, device=DEV) * (pool[0].numel() * pool.element_size())
    o = _run(dict(q=q, qo_indptr=i32([0, new]), kv_ptrs=ptrs, kv_indptr=i32([0, len(table)]),
                  last_page_offset=i32([(L - 1) % P + 1]), num_layers=1, layer_idx=0, num_kv_heads=1, base=BASE, page_size=P))

    def attend(rot):
        kr, qr = rot(k, pos)[:, 0], rot(q, pos[-new:])[:, 0]
        seen = pos[None] <= pos[-new:, None]
        e = torch.where(seen, torch.exp(qr @ kr.t() / math.sqrt(128)), 0.0)
        p = e / (e.sum(1, keepdim=True) + ahead * P)
        size = (qr.abs() @ kr.abs().t() / math.sqrt(128)).amax(1, keepdim=True)
        return p @ value[:, 0].double(), p @ value[:, 0].double().abs(), size

    def single(x, at):   # the angles as products of floats
        freq = (BASE ** (-torch.arange(64, dtype=torch.float64, device=DEV) / 64)).float()
        ang = (at.float()[:, None] * freq).double()
        c, s, a, b = ang.cos()[:, None], ang.sin()[:, None], x[..., :64].double(), x[..., 64:].double()
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    want, mass, size = attend(lambda x, at: R.rotate(x.double(), at, BASE))
    d = (2 * u * (1 + u) + 2.0 ** -13) * size
    bound = u * want.abs() + (u + torch.expm1(2 * d) + 2.0 ** -15) * mass
    err, other = (o[:, 0].double() - want).abs(), (attend(single)[0] - want).abs()
    assert (err <= bound).all(), f"{int((err > bound).sum())} past, worst {(err / bound).max()}"
    # as a whole: a score's roundings are 0.6 u of its size at most in the root mean square
    limit = ((0.6 * u + 2.0 ** -13) * size.max() + 1.3 * u).item()
    assert (err.norm() / want.norm()).item() <= limit
    assert (other > bound).any() and (other.norm() / want.norm()).item() > 2 * limit   # what the test is for
