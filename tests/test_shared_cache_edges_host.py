"""Host side of the operators around a shared cache: refusals and what a failure leaves behind.  No GPU."""


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
