"""Plain 64-bit forms of the attention operators, with the bounds that the kernels' roundings allow.

A result in bf16 is off by at most 2^-8 of itself.  Attention rounds every p to bf16 for its product with v, so each term may be off by
2^-8 of its size, and its scores are fp32 sums of `dim` products, each off by at most dim * 2^-24 of the sum of the products'
sizes; an error e of a score changes its p by a factor exp(e), and the sum that divides it as much."""
import torch

BF16 = 2.0 ** -8
FP32 = 2.0 ** -24


def attention(q, k, v, past, scale, window):
    """q [n, heads, dim] at positions past.., k and v [length, kv_heads, dim] -> (result, bound) in 64 bits."""
    n, heads, dim = q.shape
    length, kv_heads, _ = k.shape
    group = heads // kv_heads
    q, k, v = q.double(), k.double(), v.double()
    at = torch.arange(n, device=q.device)[:, None] + past
    key = torch.arange(length, device=q.device)[None]
    seen = key <= at
    if window:
        seen &= key > at - window
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    if length == 0:
        return out, bound
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        score = torch.where(seen, q[:, h] @ kh.T * scale, -torch.inf)
        size = torch.where(seen, q[:, h].abs() @ kh.T.abs() * scale, 0.0).amax(1, keepdim=True)
        top = score.amax(1, keepdim=True)
        p = torch.where(seen, torch.exp(score - torch.where(top.isinf(), 0.0, top)), 0.0)
        total = p.sum(1, keepdim=True)
        total = torch.where(total == 0, 1.0, total)
        out[:, h] = p @ vh / total
        terms = p @ vh.abs() / total
        # (the exponent is rounded twice; the exponential is off by at most 2^-18: 2^-22 from the hardware's, 2.7e-6 from the polynomial)
        bound[:, h] = BF16 * out[:, h].abs() + terms * (BF16 + 2 * (dim + 4) * FP32 * size + 64 * FP32) + 1e-30
    return out, bound


def norm(x, weight, eps):
    x = x.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return y if weight is None else y * weight.double()


def rotate(x, position, frequencies):
    """x [tokens, heads, dim] in 64 bits -> (turned, sum of the sizes that each value is made of)."""
    half = 0 if frequencies is None else frequencies.numel()
    if half == 0:
        return x, x.abs()
    angle = (position.double()[:, None] * frequencies)[:, None]
    a, b = x[..., :half], x[..., half:2 * half]
    rest = x[..., 2 * half:]
    turned = torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), rest], -1)
    both = a.abs() + b.abs()
    return turned, torch.cat([both, both, rest.abs()], -1)


def within(got, want, bound, what=""):
    got = got.double()
    assert torch.isfinite(got).all(), f"{what}: values that are not finite"
    off = (got - want).abs() - bound
    worst = off.max().item() if off.numel() else 0.0
    assert worst <= 0.0, f"{what}: {int((off > 0).sum())} of {off.numel()} beyond the bound, worst by {worst:.3g}"
