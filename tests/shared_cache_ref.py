"""64-bit references and error bounds for the operators around a shared cache (chunk attention, head norms, page copies).

A rounding to a 16-bit type is off by at most u = finfo.eps / 2 of the value (bf16 2^-8, fp16 2^-11)."""
import math

import torch

D = 128


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def rotate(x, pos, base):
    """x [..., T, N, D] float64 at integer positions [T]."""
    half = D // 2
    ang = pos.double()[:, None] * torch.pow(torch.tensor(float(base), dtype=torch.float64, device=x.device),
                                           -torch.arange(half, dtype=torch.float64, device=x.device) / half)
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def extend(q, starts, caches, base):
    """q [rows, Nq, D]; caches: per request (keys [L, N, D], values).  Returns the result in float64 (NaN in rows of no
    request) and an elementwise bound on the error of a kernel that rounds rotated queries and keys, weights and results to
    the type of q and does the rest in fp32:

    * results: u |o|;  weights: u sum p |v|
    * queries and keys: a score is off by at most d = 2 u sum |q_i k_i| / sqrt(D), a softmax weight then by a factor
      within e^(+-2 d), the result by (e^(2 d) - 1) sum p |v|
    * fp32: scores and exponentials are good to 2^-20 (|score| <= 16) or so, sums of a few thousand terms to 2^-17."""
    u = unit(q.dtype)
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for b, (K, V) in enumerate(caches):
        t0, t1 = starts[b], starts[b + 1]
        n, L = t1 - t0, K.size(0)
        if n == 0:
            continue
        G = q.size(1) // K.size(1)
        pos = torch.arange(L - n, L, device=q.device)
        qr = rotate(q[t0:t1].double(), pos, base)
        kr = rotate(K.double(), torch.arange(L, device=q.device), base)
        seen = torch.arange(L, device=q.device)[None, :] <= pos[:, None]
        for h in range(q.size(1)):
            k, v = kr[:, h // G], V[:, h // G].double()
            s = (qr[:, h] @ k.t() / math.sqrt(D)).masked_fill(~seen, -math.inf)
            size = (qr[:, h].abs() @ k.abs().t() / math.sqrt(D)).masked_fill(~seen, 0.0)
            e = torch.exp(s - s.amax(1, keepdim=True).clamp_min(-1e300))
            den = e.sum(1, keepdim=True)
            p = torch.where(den > 0, e / den, 0.0)
            o = p @ v
            mass = p @ v.abs()
            d = 2 * u * (1 + u) * size.amax(1, keepdim=True) if L else size.new_zeros((n, 1))
            out[t0:t1, h] = o
            bound[t0:t1, h] = u * o.abs() + (u + torch.expm1(2 * d) + 2.0 ** -15) * mass + 1e-30
    return out, bound


def check_extend(got, want, bound, dtype, what=""):
    """Every element within its bound; and the error as a whole: the four roundings are independent and each is 0.42 u of
    a value in the root mean square (uniform within half a step of a binary digit), so 0.84 u together; 1.3 u is allowed."""
    rows = ~torch.isnan(want).flatten(1).any(1)
    g, w = got.double()[rows], want[rows]
    assert torch.isfinite(g).all(), f"{what}: non-finite values"
    over = ((g - w).abs() > bound[rows]).sum()
    assert int(over) == 0, f"{what}: {int(over)} elements past their bound, largest excess {((g - w).abs() - bound[rows]).max()}"
    if w.numel() >= 4096:
        rel = ((g - w).norm() / w.norm()).item()
        assert rel <= 1.3 * unit(dtype), f"{what}: relative error {rel:.3g}, allowed {1.3 * unit(dtype):.3g}"


def head_norm(x, w, eps):
    """n = x rsqrt(mean x^2 + eps) w in float64."""
    x = x.double()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()


def norm_rope(x, w, pos, base, eps):
    n = x.double() if w is None else head_norm(x, w, eps)
    return n if pos is None else rotate(n, pos, base)


def norm_rope_bound(x, w, pos, base, eps, dtype):
    """u of the result, and fp32: the norm's factor, products and the sine are good to 2^-18 of the pair's size."""
    n = x.double() if w is None else head_norm(x, w, eps)
    pair = n[..., :D // 2].abs() + n[..., D // 2:].abs()
    y = norm_rope(x, w, pos, base, eps)
    return unit(dtype) * (1 + unit(dtype)) * y.abs() + 2.0 ** -18 * torch.cat([pair, pair], -1) + smallest(dtype)


def smallest(dtype):
    """Half of the smallest step of the type (fp16 values below 6e-5 are stored in steps of 6e-8)."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def norm_rope_grads(x, w, pos, g, base, eps):
    """dx, dw from the formula, in float64, and the sum of the absolute values of the terms of dw."""
    dn = g.double() if pos is None else rotate(g.double(), -pos, base)
    if w is None:
        return dn, None, None
    x, w = x.double(), w.double()
    s = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    terms = x * s * dn
    dx = s * (w * dn - x * s * s * (w * dn * x).mean(-1, keepdim=True))
    return dx, terms.sum((0, 1)), terms.abs().sum((0, 1))
