"""Host side of the operators around a shared cache: refusals and what a failure leaves behind.  No GPU."""
import pytest
import torch

import shared_cache_ref as R
from extend_whole import check_whole


def test_results_that_overlap_the_queries_are_refused():
    """Any common byte, from either side, with everything else in order; refused before any CUDA call."""
    from loquetier_b200 import cabi
    rows, heads = 8, 32
    nbytes, q = rows * heads * 128 * 2, 1 << 20
    ws = cabi.lib.smlm_b200_batch_extend_workspace_bytes(2, rows, 64, 16, heads, 8)

    def ext(o):
        return cabi.lib.smlm_b200_batch_extend(o, q, 256, 256, 256, 256, 256, ws, None, 2, rows, 64, heads, 8, 128, 1, 0, 16,
                                               10000.0, 1, None)

    for o in (q, q + 16, q - 16, q + 256, q + nbytes - 16, q - nbytes + 16):
        assert ext(o) == 1


@pytest.mark.parametrize("fails", ["slab", "table"])
def test_a_cache_that_cannot_be_made_keeps_no_pages(monkeypatch, fails):
    """The memory ends at the third slab, or at the table of addresses: the pages taken so far are free again, and their slabs
    can be given back."""
    from loquetier_b200 import kvcache
    pool = kvcache.KvPool(1, 1, 8, 4, torch.float32, "cpu", pages_per_slab=2)
    kept = kvcache.KvCache(pool, 5)
    real, slabs = torch.empty, []

    def empty(*a, **kw):
        slabs.append(1)
        if len(slabs) == 3:
            raise RuntimeError("out of memory")
        return real(*a, **kw)

    def table(*a, **kw):
        raise RuntimeError("out of memory")

    if fails == "slab":
        monkeypatch.setattr(torch, "empty", empty)
    else:
        monkeypatch.setattr(kvcache, "GrowableTensor", table)
    with pytest.raises(RuntimeError, match="out of memory"):
        kvcache.KvCache(pool, 30)
    monkeypatch.undo()
    assert pool.num_pages == 2 and [p.data_ptr() for p in pool.allocated_pages()] == [p.data_ptr() for p in kept.pages]
    assert len(pool._free) == pool.num_slabs * 2 - 2
    kept.release()
    assert pool.compact([kept]) and pool.num_slabs == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [(8, 4), (1, 8), (3, 1), (1, 1)])
@pytest.mark.parametrize("new,length", [(1, 5003), (2, 5003), (7, 9001)])
def test_the_check_as_a_whole_rejects_what_is_lost(dtype, heads, new, length):
    """For few rows over many keys the elementwise bounds let a zero pass; the check of the whole result does not, nor a
    share of 4 tiles of 64 keys that is lost or counted twice.  Roundings pass."""
    (N, G), cut = heads, slice(256, 512)
    g = torch.Generator().manual_seed(new)
    q = torch.randn((new, N * G, 128), generator=g).to(dtype)
    K, V = (torch.randn((length, N, 128), generator=g).to(dtype) for _ in range(2))
    want, _ = R.extend(q, [0, new], [(K, V)], 1e4)
    check_whole(want.to(dtype), want, dtype)

    def attend(weight):   # keys counted so often, in 64 bits
        pos = torch.arange(length)
        kr, qr = R.rotate(K.double(), pos, 1e4), R.rotate(q.double(), pos[-new:], 1e4)
        s = torch.einsum("nhgd,lhd->nhgl", qr.unflatten(1, (N, G)), kr) / 128 ** 0.5
        e = torch.exp(s) * weight * (pos[None] <= pos[-new:, None]).double()[:, None, None]
        return torch.einsum("nhgl,lhd->nhgd", e / e.sum(-1, keepdim=True), V.double()).flatten(1, 2)

    weight = torch.ones(length, dtype=torch.float64)
    check_whole(attend(weight).to(dtype), want, dtype)
    for wrong in (0.0, 2.0):
        weight[cut] = wrong
        with pytest.raises(AssertionError):
            check_whole(attend(weight), want, dtype)
    with pytest.raises(AssertionError):
        check_whole(torch.zeros_like(want), want, dtype)


def test_the_backward_asks_first_whether_a_capture_runs(monkeypatch):
    """Without a GPU: nothing of the saved tensors is used before the refusal."""
    from types import SimpleNamespace

    from loquetier_b200 import ops
    from loquetier_b200.kernel_utils import qk_norm_rope

    def refuse(t, what):
        raise RuntimeError(f"{what} cannot be captured")

    monkeypatch.setattr(ops, "refuse_capture", refuse)
    ctx = SimpleNamespace(saved_tensors=(None,) * 5)   # anything done with them would raise something else
    with pytest.raises(RuntimeError, match="the backward of qk_norm_rope cannot be captured"):
        qk_norm_rope.backward(ctx, None, None)
