"""Plain forms of the layer operators in 64 bits, and the same steps in fp32 where the definition names every rounding."""
import torch

U = 2.0 ** -24
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def norm(x, weight, variant, eps):
    """In 64 bits."""
    if variant == -1:
        return x
    x = x / torch.sqrt((x * x).mean(1, keepdim=True) + eps)
    return x if variant == 2 else x * (weight.double() + (1.0 if variant == 1 else 0.0))


def add_norm(h, y, weight, variant, post_weight, post_variant, gate, alpha, eps):
    """(p, h', n) in 64 bits."""
    p = torch.zeros_like(h.double()) if y is None else norm(y.double(), post_weight, post_variant, eps)
    if gate is not None:
        p = p * gate.double()
    p = p * float(torch.tensor(alpha, dtype=torch.float32))
    s = h.double() + p
    return p, s, norm(s, weight, variant, eps)


def norm32(x, weight, variant, eps):
    """The definition's fp32 steps: the factor taken in 64 bits and rounded, then one product after the other."""
    if variant == -1:
        return x
    r = (1.0 / torch.sqrt((x.double() ** 2).sum(1, keepdim=True) / x.shape[1] + eps)).float()
    x = x * r
    return x if variant == 2 else x * (weight if variant == 0 else 1.0 + weight)


def add_norm32(h, y, weight, variant, post_weight, post_variant, gate, alpha, eps):
    s = h.float()
    if y is not None:
        p = norm32(y.float(), post_weight, post_variant, eps)
        p = p if gate is None else p * gate
        s = s + p * torch.tensor(alpha, dtype=torch.float32, device=s.device)
    return s, norm32(s, weight, variant, eps)


def quantize(x, group):
    """fp32 rows to codes, scales and sums of blocks of `group` elements (0: whole rows); every step is an fp32 operation."""
    S, K = x.shape
    b = x.view(S, 1 if group == 0 else K // group, -1)
    scale = b.abs().amax(2) / torch.tensor(127.0, device=x.device)
    q = torch.where(scale[..., None] > 0, torch.round(b / scale[..., None]), torch.zeros_like(b)).clamp(-127, 127).to(torch.int8)
    return q.view(S, K), scale, q.sum(2, dtype=torch.int32)


def near(got, want, slack, what):
    """|got - want| <= slack + half a step of got's type, everywhere."""
    info = torch.finfo(got.dtype)
    half = want.abs() * (info.eps / 2) + float(info.smallest_normal) * info.eps / 2
    off = (got.double() - want).abs() - (slack + half)
    assert torch.isfinite(got).all() and (off <= 0).all(), (what, float(off.max()), int((off > 0).sum()))
