"""``qk_norm_rope`` without an epsilon, and its backward under capture.  Bounds: as in ``test_gpu_head_norm``."""
import pytest
import torch

import shared_cache_ref as R
from test_gpu_head_norm import BASE, DEV, EPS, _inputs, _within

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


def test_the_backward_itself_is_refused_under_capture():
    """The node's backward, on what its forward saved, while a capture runs: refused before it allocates or launches, and
    the same call answers outside."""
    from types import SimpleNamespace

    from loquetier_b200.kernel_utils import qk_norm_rope
    q, k, _, wq, wk, gq, gk = _inputs(7, 5, 4, 2, torch.bfloat16)
    pos = torch.arange(5, device=DEV)
    args = [t.detach().clone().requires_grad_() for t in (q, k, wq, wk)]
    want = torch.autograd.grad(qk_norm_rope.apply(*args, pos, BASE, EPS), args, (gq, gk))
    saved = [t.detach() for t in args]
    ctx = SimpleNamespace(saved_tensors=(*saved, pos), base=BASE, eps=EPS, strides=(4 * 128, 2 * 128),
                          needs_input_grad=(True, True, True, True, False, False, False))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph, seen = torch.cuda.CUDAGraph(), torch.zeros(1, device=DEV)
    with torch.cuda.graph(graph, stream=stream):
        seen += 1
        held = torch.cuda.memory_allocated()
        with pytest.raises(RuntimeError, match="the backward of qk_norm_rope cannot be captured"):
            qk_norm_rope.backward(ctx, gq, gk)
        assert torch.cuda.memory_allocated() == held
    graph.replay()
    got = qk_norm_rope.backward(ctx, gq, gk)
    torch.cuda.synchronize()
    assert seen.item() == 1 and all(torch.equal(a, b) for a, b in zip(got, want))
