"""``kvcache.batch_extend`` at the edges of its range."""
import pytest
import torch

from test_gpu_batch_extend import DEV, LAYER, _batch, _run

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
