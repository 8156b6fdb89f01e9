"""Host side of the operators around a shared cache: refusals and what a failure leaves behind.  No GPU."""
import pytest
import torch


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
