"""Values in 4 bits for the tests: the format's formulas in plain tensors."""
import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # of rounding


def quantised(x, group):
    """Codes (float64) and (step, low) pairs, in the type of x, of the last dimension's groups; NaN pairs where a value is not
    finite, a step of 0 where all are alike."""
    g = x.unflatten(-1, (-1, group)).double()
    low, top = g.amin(-1), g.amax(-1)
    step = ((top - low).float() / 15).to(x.dtype)
    bad = ~torch.isfinite(g).all(-1) | ~torch.isfinite(step)
    s = step.double()[..., None]
    codes = torch.where(s > 0, ((g - low[..., None]).float() / s.float()).double(), 0.0).round().clamp(0, 15)
    codes = torch.where(bad[..., None], 0.0, codes.nan_to_num(0.0))
    nan = torch.full_like(step, float("nan"))
    return codes.flatten(-2), torch.stack([torch.where(bad, nan, step), torch.where(bad, nan, low.to(x.dtype))], -1)


def values(codes, scales, group):
    """What they stand for, in 64 bits; the last group may be short."""
    s = scales.double().repeat_interleave(group, -2)[..., :codes.shape[-1], :]
    return s[..., 1] + s[..., 0] * codes.double()


def held(x, group):
    return values(*quantised(x, group), group)


def packed_pairs(codes):
    """Two columns a byte, the even one's in the low half."""
    c = codes.to(torch.uint8)
    return (c[..., 0::2] | c[..., 1::2] << 4).contiguous()


def randn(seed, *shape, dtype=torch.bfloat16, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(*shape, device="cuda", generator=g)).to(dtype)


def by_heads(x, heads):
    """(B, rows, heads * hd) -> (B, heads, rows, hd)"""
    return x.unflatten(-1, (heads, -1)).transpose(1, 2)


def flat(x):
    return x.transpose(1, 2).flatten(-2)
