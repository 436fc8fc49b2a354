"""Groups of 32 with values next to a border between two codes (test only).

With a = x - b, a value lies on a border where a = (k + 1/2) s.  Where |x| is far below |b|, fp32
rounds a, and may round it onto a border that it does not lie on: then the nearest code is the one on
x's own side.  `groups` finds ends of a group whose -b lies next to a border, and fills it with such
values."""
import torch


def groups(dtype, count, seed=0):
    """[count, 32] of dtype: two ends, and values x with fp32(x - b) on a border, x - b not."""
    g = torch.Generator().manual_seed(seed)
    found, have = [], 0
    while have < count:
        n = 400000
        lo = (-0.5 - 2 * torch.rand(n, generator=g, dtype=torch.float64)).to(dtype).double()
        hi = (0.5 + 2 * torch.rand(n, generator=g, dtype=torch.float64)).to(dtype).double()
        s = ((hi - lo) / 15).to(dtype).double()
        b = (lo - 16 * s).to(dtype).double()
        border = (torch.floor(-b / s) + 0.5) * s + b  # the x that lies on the border next to 0
        rows = border.abs() < b.abs() * (2.0 ** -13 if dtype == torch.float16 else 2.0 ** -16)
        lo, hi, s, b, border = (x[rows] for x in (lo, hi, s, b, border))
        # Numbers of the type within half a unit of fp32 in b of the border, and not on it.
        unit = torch.exp2(torch.floor(torch.log2(b.abs())) - 23)
        x = (border[:, None] + unit[:, None] * torch.linspace(-0.49, 0.49, 30,
                                                              dtype=torch.float64)).to(dtype).double()
        a = x - b[:, None]
        hit = (a.float().double() == border[:, None] - b[:, None]) & (x != border[:, None])
        x = torch.where(hit, x, 0.0)
        keep = hit.any(-1)
        out = torch.cat([lo[:, None], hi[:, None], x], -1)[keep].to(dtype)
        found.append(out)
        have += out.shape[0]
    return torch.cat(found)[:count]
