"""The 8-bit codes from their definition in fp64, for the tests (no code of the package)."""
import torch


def nearest(t):
    """The whole number nearest to t, the even one of two that are as near."""
    low = torch.floor(t)
    rest = t - low
    return low + ((rest > 0.5) | ((rest == 0.5) & (torch.remainder(low, 2) == 1))).double()


def rows(x):
    """(codes, scales) in fp64 of x [R, K] with one scale a row: NaN scales and codes of 0 where a row is not finite."""
    x = x.double()
    size = x.abs().amax(1)
    bad = ~torch.isfinite(x).all(1)
    size = torch.where(bad, torch.zeros_like(size), size)
    s = torch.clamp((size.float() / 127).double(), min=2.0 ** -126, max=float.fromhex("0x1.020406p121"))  # 127 times that is finite
    s = torch.where(size > 0, s, torch.ones_like(s))
    c = torch.where(bad[:, None], torch.zeros_like(x), nearest(torch.where(bad[:, None], torch.zeros_like(x), x) / s[:, None]))
    return c, torch.where(bad, torch.full_like(s, float("nan")), s)


def blocks(x):
    """(codes, exponents plus 127) in fp64 of x [R, K] in blocks of 32 columns."""
    R, K = x.shape
    xb = torch.nn.functional.pad(x.double(), (0, -K % 32)).reshape(R, (K + 31) // 32, 32)
    bad = ~torch.isfinite(xb).all(2)
    xb = torch.where(bad[..., None], torch.zeros_like(xb), xb)
    top = xb.abs().amax(2)
    e = torch.frexp(top)[1].double() - 1 - 6  # frexp's mantissa is in [1/2, 1)
    e = torch.where(top > 0, e, torch.full_like(e, -127)).clamp(min=-127)
    # x / 2^e in two steps, each exact in fp64
    c = nearest(torch.ldexp(xb, -e[..., None])).clamp(-127, 127)
    return c.reshape(R, -1)[:, :K], torch.where(bad, torch.full_like(e, 255.0), e + 127)


def values(x, block):
    """What x's codes stand for, in fp64."""
    if block == 0:
        c, s = rows(x)
        return c * s[:, None]
    c, e = blocks(x)
    s = torch.where(e == 255, torch.full_like(e, float("nan")), torch.ldexp(torch.ones_like(e), e - 127))
    return c * s.repeat_interleave(32, dim=1)[:, :x.shape[1]]
