"""``batch_prefill`` on chunks: a few new tokens per request behind a long cache.  Most rows of a tile then do not exist and
their softmax warps run ahead of those that raise their maxima; no wait may run out, and the results hold."""
import pytest
import torch

import shared_cache_ref as R
from test_gpu_batch_extend import BASE, LAYER, LAYERS, _batch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("group,new,length", [(4, 5, 2500), (1, 60, 2100), (8, 1, 3000), (2, 17, 900)])
def test_prefill_of_chunks_behind_long_caches(group, new, length):
    from loquetier_b200 import kvcache
    lens, runs = [length - 13 * i for i in range(12)], [max(1, new - i % 3) for i in range(12)]
    pool, args, starts, dense = _batch(group + new, lens, runs, 4, group, 16, torch.bfloat16, poison=False)
    q = args["q"][:starts[-1]].contiguous()
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    for _ in range(5):
        o = torch.full_like(q, 7.0)
        kvcache.batch_prefill_into(o, q, args["qo_indptr"], args["kv_ptrs"], args["kv_indptr"], args["last_page_offset"],
                                   LAYERS, LAYER, 4, BASE, 16, status_word=word)
        torch.cuda.synchronize()
        assert int(word.item()) == 0
        want, bound = R.extend(q, starts, dense, BASE)
        # (the angles are single precision there: 2^-11 of a radian at these positions, of scores of order one)
        assert ((o.double() - want).norm() / want.norm()).item() <= 1.6 * R.unit(torch.bfloat16)
