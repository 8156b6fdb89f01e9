"""``qk_norm_rope`` without an epsilon, and its backward under capture.  Bounds: as in ``test_gpu_head_norm``."""
import pytest
import torch

import shared_cache_ref as R
from test_gpu_head_norm import BASE, DEV, _inputs, _within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rope", [True, False])
@pytest.mark.parametrize("T,Nq,Nk", [(1, 1, 1), (3, 2, 1), (9, 5, 2), (70, 6, 5), (1200, 7, 3), (33, 8, 4)])
def test_gradients_without_epsilon(dtype, rope, T, Nq, Nk):
    """eps = 0: rows without zeros have finite gradients, whatever the number of heads - a warp works on four at a time, and
    the places behind the last head must not count."""
    from loquetier_b200.kernel_utils import qk_norm_rope
    q, k, _, wq, wk, gq, gk = _inputs(T + Nq, T, Nq, Nk, dtype)
    pos = torch.arange(T, device=DEV) * 3 + 1 if rope else None
    args = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    yq, yk = qk_norm_rope.apply(*args, pos, BASE, 0.0)
    grads = torch.autograd.grad((yq, yk), args, (gq, gk))
    u = R.unit(dtype)
    for i, (x, w, y, g) in enumerate(((q, wq, yq, gq), (k, wk, yk, gk))):
        _within(y.detach(), R.norm_rope(x, w, pos, BASE, 0.0), R.norm_rope_bound(x, w, pos, BASE, 0.0, dtype), f"y{i}")
        dx, dw, terms = R.norm_rope_grads(x, w, pos, g, BASE, 0.0)
        dn = R.norm_rope_grads(x, None, pos, g, BASE, 0.0)[0]
        pair = dn[..., :64].abs() + dn[..., 64:].abs()
        size = torch.cat([pair, pair], -1)
        x64, w64 = x.double(), w.double()
        s = torch.rsqrt((x64 * x64).mean(-1, keepdim=True))
        pair_terms = ((x64 * s).abs() * size).sum((0, 1))
        size = s * (w64.abs() * size + x64.abs() * s * s * (w64.abs() * size * x64.abs()).mean(-1, keepdim=True))
        _within(grads[i], dx, u * (1 + u) * dx.abs() + 2.0 ** -18 * size + R.smallest(dtype), f"dx{i}")
        _within(grads[2 + i], dw, u * (1 + u) * dw.abs() + 2.0 ** -18 * pair_terms + 2.0 ** -14 * terms + R.smallest(dtype),
                f"dw{i}")
