"""Norms of queries and keys per head: with the rotation for trained rows (``kernel_utils.qk_norm_rope``) and into the pages for
served ones (``kvcache.norm_append_kv``), against their definition in 64 bits with bounds by arithmetic."""
import pytest
import torch

import shared_cache_ref as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BASE, EPS = 10000.0, 1e-6


def _inputs(seed, T, Nq, Nk, dtype, scale=1.7):
    g = torch.Generator(device=DEV).manual_seed(seed)
    qkv = (torch.randn((T, Nq + 2 * Nk, 128), generator=g, device=DEV) * scale).to(dtype)
    w = lambda: (1 + 0.3 * torch.randn(128, generator=g, device=DEV)).to(dtype)
    grad = lambda n: torch.randn((T, n, 128), generator=g, device=DEV).to(dtype)
    return qkv[:, :Nq], qkv[:, Nq:Nq + Nk], qkv[:, Nq + Nk:], w(), w(), grad(Nq), grad(Nk)


def _within(got, want, bound, what):
    d = (got.double() - want).abs()
    assert torch.isfinite(got).all() and (d <= bound).all(), f"{what}: {int((d > bound).sum())} past, worst {(d / bound).max()}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("norm,rope", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("T,Nq,Nk", [(1, 32, 8), (1, 1, 1), (2, 5, 3), (7, 8, 8), (33, 32, 8), (301, 4, 1), (2500, 6, 2)])
def test_forward_and_backward(dtype, norm, rope, T, Nq, Nk):
    from loquetier_b200.kernel_utils import qk_norm_rope
    q, k, _, wq, wk, gq, gk = _inputs(T + Nq, T, Nq, Nk, dtype)
    if not norm:
        wq = wk = None
    pos = (torch.arange(T, device=DEV, dtype=torch.int64 if T % 2 else torch.int32) * 37 + 5) if rope else None
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk) if t is not None]
    args = [t.detach().requires_grad_() if t is not None else None for t in (q, k, wq, wk)]
    yq, yk = qk_norm_rope.apply(*args, pos, BASE, EPS)
    assert yq.is_contiguous() and yk.is_contiguous()
    grads = torch.autograd.grad((yq, yk), [a for a in args if a is not None], (gq, gk))
    again = torch.autograd.grad(qk_norm_rope.apply(*args, pos, BASE, EPS), [a for a in args if a is not None], (gq, gk))
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    for i, (x, w, y, g) in enumerate(((q, wq, yq, gq), (k, wk, yk, gk))):
        _within(y.detach(), R.norm_rope(x, w, pos, BASE, EPS), R.norm_rope_bound(x, w, pos, BASE, EPS, dtype), f"y{i}")
        dx, dw, terms = R.norm_rope_grads(x, w, pos, g, BASE, EPS)
        # u of the result; fp32 and the sine, 2^-18 of what is added: s (|w dn| + |x| s^2 mean |w dn x|), a pair's dn
        dn = R.norm_rope_grads(x, None, pos, g, BASE, EPS)[0]
        pair = dn[..., :64].abs() + dn[..., 64:].abs()
        size = torch.cat([pair, pair], -1)
        if norm:
            x64, w64 = x.double(), w.double()
            s = torch.rsqrt((x64 * x64).mean(-1, keepdim=True) + EPS)
            size = s * (w64.abs() * size + x64.abs() * s * s * (w64.abs() * size * x64.abs()).mean(-1, keepdim=True))
        u = R.unit(dtype)
        _within(grads[i], dx, u * (1 + u) * dx.abs() + 2.0 ** -18 * size + R.smallest(dtype), f"dx{i}")
        if norm:   # each term as above, then an fp32 sum whose partial sums hold at most 2^10 terms in a row: 2^-14
            x_s = (x.double() * torch.rsqrt((x.double() ** 2).mean(-1, keepdim=True) + EPS)).abs()
            pair_terms = (x_s * torch.cat([pair, pair], -1)).sum((0, 1))
            _within(grads[2 + i], dw, u * (1 + u) * dw.abs() + 2.0 ** -18 * pair_terms + 2.0 ** -14 * terms + R.smallest(dtype),
                    f"dw{i}")


def test_far_positions_lose_nothing():
    """At 200 000 and at 2^24 - 1 a single-precision angle would be off by hundredths of a radian and more."""
    from loquetier_b200.kernel_utils import qk_norm_rope
    q, k, _, wq, wk, _, _ = _inputs(3, 64, 4, 2, torch.float16)
    for first in (200000, (1 << 24) - 64):
        pos = torch.arange(first, first + 64, device=DEV)
        yq, yk = qk_norm_rope.apply(q, k, wq, wk, pos, 500000.0, EPS)
        _within(yq, R.norm_rope(q, wq, pos, 500000.0, EPS), R.norm_rope_bound(q, wq, pos, 500000.0, EPS, torch.float16), "far")


def test_extreme_rows():
    """Rows of zeros stay zeros and pass a finite gradient; large and tiny rows do not overflow on the way; a NaN stays in
    its head."""
    from loquetier_b200.kernel_utils import qk_norm_rope
    q, k, _, wq, wk, gq, gk = _inputs(4, 6, 4, 4, torch.bfloat16)
    q = q.clone()
    q[0] = 0
    q[1] *= 1e15
    q[2] *= 1e-12
    q[3, 1, 7] = float("nan")
    q.requires_grad_()
    yq, _ = qk_norm_rope.apply(q, k, wq, wk, None, BASE, EPS)
    assert (yq[0] == 0).all() and torch.isnan(yq[3, 1]).all()
    keep = torch.ones((6, 4), dtype=torch.bool, device=DEV)
    keep[3, 1] = False
    assert torch.isfinite(yq[keep]).all()
    want = R.norm_rope(q.detach(), wq, None, BASE, EPS)
    bound = R.norm_rope_bound(q.detach(), wq, None, BASE, EPS, torch.bfloat16)
    assert ((yq.detach().double() - want).abs() <= bound)[keep].all()
    dq, = torch.autograd.grad(yq, q, gq)
    assert torch.isfinite(dq[keep]).all()


def test_no_rows_and_unused_outputs():
    from loquetier_b200.kernel_utils import qk_norm_rope
    q, k, _, wq, wk, gq, _ = _inputs(5, 3, 4, 2, torch.bfloat16)
    e = [q[:0].detach().requires_grad_(), k[:0].detach().requires_grad_(), wq.requires_grad_(), wk.requires_grad_()]
    yq, yk = qk_norm_rope.apply(*e, None, BASE, EPS)
    g = torch.autograd.grad((yq.sum() + yk.sum()), e)
    assert all((t == 0).all() for t in g)
    # only the queries are used: the keys' gradients are zeros
    args = [q.detach().requires_grad_(), k.detach().requires_grad_(), wq, wk]
    yq, _ = qk_norm_rope.apply(*args, torch.arange(3, device=DEV), BASE, EPS)
    dq, dk, _, dwk = torch.autograd.grad(yq, args, gq)
    assert (dk == 0).all() and (dwk == 0).all() and (dq != 0).any()


def test_gradients_of_broadcast_and_transposed_outputs():
    """Gradients arrive as autograd makes them: expanded, transposed.  A head of keys that all query heads share."""
    from loquetier_b200.kernel_utils import qk_norm_rope
    q, k, _, wq, wk, _, _ = _inputs(6, 9, 4, 1, torch.float16)
    args = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    yq, yk = qk_norm_rope.apply(*args, torch.arange(9, device=DEV), BASE, EPS)
    loss = (yq.float().transpose(0, 1) * yk.float().expand(9, 4, 128).transpose(0, 1)).sum()
    got = torch.autograd.grad(loss, args)
    x = [t.detach().double().requires_grad_() for t in (q, k, wq, wk)]
    pos = torch.arange(9, device=DEV)
    want = torch.autograd.grad((R.norm_rope(x[0], x[2], pos, BASE, EPS) * R.norm_rope(x[1], x[3], pos, BASE, EPS)).sum(), x)
    # the gradients that reach the kernel are themselves rounded outputs of it: two roundings more, of the largest value
    for a, b in zip(got, want):
        assert (a.double() - b).abs().max() <= 4 * R.unit(torch.float16) * 8 * b.abs().max()


@pytest.mark.parametrize("T", [1, 77])
def test_weights_that_are_not_trained(T):
    """Their gradients are not formed; the others are the same bits.  One of them alone may be trained."""
    from loquetier_b200.kernel_utils import qk_norm_rope
    q, k, _, wq, wk, gq, gk = _inputs(8, T, 8, 2, torch.bfloat16)
    pos = torch.arange(T, device=DEV)
    x = [t.detach().clone().requires_grad_() for t in (q, k)]
    w = [t.detach().clone().requires_grad_() for t in (wq, wk)]
    want = torch.autograd.grad(qk_norm_rope.apply(*x, *w, pos, BASE, EPS), x + w, (gq, gk))
    got = torch.autograd.grad(qk_norm_rope.apply(*x, wq.detach(), wk.detach(), pos, BASE, EPS), x, (gq, gk))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = torch.autograd.grad(qk_norm_rope.apply(*x, wq.detach(), w[1], pos, BASE, EPS), x + w[1:], (gq, gk))
    assert all(torch.equal(a, b) for a, b in zip(got, want[:2] + want[3:]))


def test_offsets_past_32_bits():
    """2^31 elements and more: the last rows are the bits that a call of their own gives, in both directions."""
    from loquetier_b200.kernel_utils import qk_norm_rope
    T, Nq, Nk, n = (1 << 31) // (64 * 128) + 5, 64, 1, 9
    q = torch.empty((T, Nq, 128), dtype=torch.bfloat16, device=DEV)
    k = torch.empty((T, Nk, 128), dtype=torch.bfloat16, device=DEV)
    gq = torch.empty_like(q)
    small = _inputs(9, n, Nq, Nk, torch.bfloat16)
    for big, part in ((q, small[0]), (k, small[1]), (gq, small[5])):
        big.normal_()
        big[-n:] = part
    gk = torch.ones_like(k)
    pos = torch.arange(T, device=DEV)
    wq, wk = small[3], small[4]
    args = [q.requires_grad_(), k.requires_grad_()]
    y = qk_norm_rope.apply(*args, wq, wk, pos, BASE, EPS)
    tail = [t.detach()[-n:].clone().requires_grad_() for t in args]
    ty = qk_norm_rope.apply(*tail, wq, wk, pos[-n:].contiguous(), BASE, EPS)
    assert all(torch.equal(a[-n:], b) for a, b in zip(y, ty))
    got = torch.autograd.grad(y, args, (gq, gk))
    want = torch.autograd.grad(ty, tail, (gq[-n:].contiguous(), gk[-n:].contiguous()))
    assert all(torch.equal(a[-n:], b) for a, b in zip(got, want))


def test_backward_under_capture_is_refused():
    from loquetier_b200.kernel_utils import qk_norm_rope
    q, k, _, wq, wk, gq, gk = _inputs(7, 5, 4, 2, torch.bfloat16)
    args = [t.detach().clone().requires_grad_() for t in (q, k, wq, wk)]
    pos = torch.arange(5, device=DEV)
    want = qk_norm_rope.apply(*args, pos, BASE, EPS)
    from loquetier_b200 import ops
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):     # a forward can be captured
        got = qk_norm_rope.apply(*[a.detach() for a in args], pos, BASE, EPS)
        with pytest.raises(RuntimeError, match="cannot be captured"):
            ops.refuse_capture(q, "the backward of qk_norm_rope")
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------
# into the cache
# ---------------------------------------------------------------------------

def _cache(lens, N, P, dtype, layers=2):
    from loquetier_b200 import kvcache
    pool = kvcache.KvPool(layers, N, 128, P, dtype, DEV, pages_per_slab=4)
    caches = [kvcache.KvCache(pool, L) for L in lens]
    for c in caches:
        for p in c.pages:
            p.fill_(7.0)
    return pool, caches, kvcache.BatchedKvCache(caches)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Nq,Nk,P", [(32, 8, 16), (5, 1, 8), (8, 8, 64), (3, 3, 32)])
@pytest.mark.parametrize("new", [None, [1, 5, 0, 40, 2], [17, 1, 1, 0, 16]])
def test_norm_append(dtype, Nq, Nk, P, new):
    from loquetier_b200 import kvcache
    lens = [20, 5, 33, 40, 16] if new is None else [max(n, 1) + e for n, e in zip(new, (3, 0, 30, 0, 65))]
    pool, caches, kv = _cache(lens, Nk, P, dtype)
    runs = [1] * 5 if new is None else new
    T = sum(runs)
    q, k, v, wq, wk, _, _ = _inputs(T, T + 2, Nq, Nk, dtype)
    if new is None:
        q, k, v, ind = q[:T], k[:T], v[:T], None
    else:
        starts = [0]
        for n in runs:
            starts.append(starts[-1] + n)
        ind = torch.tensor(starts, dtype=torch.int32, device=DEV)
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = kvcache.norm_append_kv(kv, q, k, v, wq, wk, EPS, 1, ind, status_word=word)
    torch.cuda.synchronize()
    assert int(word.item()) == 0
    _within(out[:T], R.head_norm(q[:T], wq, EPS), R.norm_rope_bound(q[:T], wq, None, BASE, EPS, dtype), "q")
    want_k, bound_k = R.head_norm(k[:T], wk, EPS), R.norm_rope_bound(k[:T], wk, None, BASE, EPS, dtype)
    t = 0
    for c, n, L in zip(caches, runs, lens):
        for i, page in enumerate(c.pages):
            assert (page[0] == 7.0).all()                      # the other layer
            for e in range(P):
                pos = i * P + e
                if L - n <= pos < L:
                    j = t + pos - (L - n)
                    assert ((page[1, 0, :, e].double() - want_k[j]).abs() <= bound_k[j]).all()
                    assert torch.equal(page[1, 1, :, e], v[j])
                else:
                    assert (page[1, :, :, e] == 7.0).all()
        t += n


def test_norm_append_equals_norm_then_append():
    """The same bits as normalising through ``qk_norm_rope`` and writing through ``init_kv``."""
    from loquetier_b200 import kvcache
    from loquetier_b200.kernel_utils import qk_norm_rope
    lens = [30, 9, 77]
    _, caches, kv = _cache(lens, 4, 16, torch.bfloat16)
    _, caches2, kv2 = _cache(lens, 4, 16, torch.bfloat16)
    q, k, v, wq, wk, _, _ = _inputs(8, 60, 16, 4, torch.bfloat16)
    ind = torch.tensor([0, 20, 25, 60], dtype=torch.int32, device=DEV)
    out = kvcache.norm_append_kv(kv, q, k, v, wq, wk, EPS, 0, ind)
    nq, nk = qk_norm_rope.apply(q, k, wq, wk, None, BASE, EPS)
    kvcache.init_kv(kv2, nk, v.contiguous(), ind, 0)
    torch.cuda.synchronize()
    assert torch.equal(out, nq)
    for a, b in zip(caches, caches2):
        assert all(torch.equal(p, r) for p, r in zip(a.pages, b.pages))


def test_norm_append_reports_what_the_pages_do_not_hold():
    from loquetier_b200 import kvcache
    _, caches, kv = _cache([5, 20], 2, 16, torch.bfloat16)
    q, k, v, wq, wk, _, _ = _inputs(9, 9, 4, 2, torch.bfloat16)
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    ind = torch.tensor([0, 6, 9], dtype=torch.int32, device=DEV)      # six new tokens in a cache of five
    out = kvcache.norm_append_kv(kv, q, k, v, wq, wk, EPS, 0, ind, status_word=word)
    torch.cuda.synchronize()
    assert int(word.item()) == 1
    assert (caches[0].pages[0] == 7.0).all() and (caches[1].pages[1][0, 1, :, 1:4] == v[6:9].transpose(0, 1)).all()
    _within(out, R.head_norm(q, wq, EPS), R.norm_rope_bound(q, wq, None, BASE, EPS, torch.bfloat16), "q")
    word.zero_()
    kv.ptrs[2] = 0
    kvcache.norm_append_kv(kv, q[:2], k[:2], v[:2], wq, wk, EPS, 0, status_word=word)
    torch.cuda.synchronize()
    assert int(word.item()) == 2
