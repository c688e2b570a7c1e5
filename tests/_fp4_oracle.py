"""64-bit oracle of the 4-bit formats: every value by search over the representable numbers, no shared code with
the package."""
import torch

LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
BLOCK = {"mxfp4": 32, "nvfp4": 16}
# e4m3 numbers >= 0 in the order of their codes 0 .. 126
E4M3 = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:119]


def nearest(v: torch.Tensor, table) -> torch.Tensor:
    """Index of the nearest number of an ascending table (halves to the even index, the last one at most)."""
    t = torch.tensor(table, dtype=torch.float64, device=v.device)
    hi = torch.searchsorted(t, v).clamp(max=len(table) - 1)
    lo = (hi - 1).clamp(min=0)
    dh, dl = (t[hi] - v).abs(), (v - t[lo]).abs()
    return torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)


def values(x: torch.Tensor, fmt: str):
    """(values fp64 [R, K], scale codes [R, blocks], row scales [R]) of the 4-bit form of rows x."""
    R, K = x.shape
    blk = BLOCK[fmt]
    x = x.double().cpu()
    out = torch.zeros(R, K, dtype=torch.float64)
    codes = torch.zeros(R, -(-K // blk), dtype=torch.long)
    row = torch.ones(R, dtype=torch.float64)
    if fmt == "nvfp4":
        fin = torch.zeros(R, dtype=torch.float64)
        for b in range(codes.shape[1]):
            a = x[:, b * blk:(b + 1) * blk].abs().amax(1)
            fin = torch.maximum(fin, torch.where(torch.isfinite(a), a, 0.0))
        g = torch.full((R,), 2.0 ** -126, dtype=torch.float64)
        for _ in range(300):
            g = torch.where(fin > 2688.0 * g, 2 * g, g)
        row = torch.where(fin > 0, g, 1.0)
    for b in range(codes.shape[1]):
        xb = x[:, b * blk:(b + 1) * blk]
        a = xb.abs().amax(1)
        bad = ~torch.isfinite(a)
        a = torch.where(bad, 0.0, a)
        if fmt == "mxfp4":
            e = torch.full((R,), -127.0, dtype=torch.float64)
            for _ in range(254):
                e = torch.where(a >= torch.exp2(e + 3), e + 1, e)
            c, s = (e + 127).long(), torch.exp2(e)
            nan = 255
        else:
            c = nearest(a / row / 6, E4M3)
            s = torch.tensor(E4M3, dtype=torch.float64)[c] * row
            nan = 127
        v = torch.where(s[:, None] > 0, torch.where(bad[:, None], 0.0, xb.abs()) / s[:, None], 0.0)
        q = torch.tensor(LEVELS, dtype=torch.float64)[nearest(v, LEVELS)] * s[:, None]
        out[:, b * blk:(b + 1) * blk] = torch.where(bad[:, None], float("nan"), torch.where(xb < 0, -q, q))
        codes[:, b] = torch.where(bad, nan, c)
    return out, codes, row


def inputs(R, K, dtype, seed=0, kind="normal"):
    """normal: rows of different sizes; grid: short significands, so halves and block maxima on borders are common."""
    g = torch.Generator().manual_seed(seed)
    if kind == "normal":
        x = torch.randn(R, K, generator=g) * torch.exp(2 * torch.randn(R, 1, generator=g))
    else:
        x = torch.randint(-28, 29, (R, K), generator=g) * 0.25 * 2.0 ** torch.randint(-6, 7, (R, K // 16 + 1),
                                                                                     generator=g).repeat_interleave(16, 1)[:, :K]
    return x.to(dtype)
