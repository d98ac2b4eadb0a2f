"""Plain 64-bit forms of the power-of-two block-scaled operators, on the CPU, for the tests."""
import torch

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def quantize(x, square=False):
    """(codes as uint8, scale bytes as uint8 [blocks of columns, rows or blocks of rows]) of x along its rows."""
    rows, cols = x.shape
    x = x.detach().cpu().double()
    step = 128 if square else 1
    nr, nc = -(-rows // step), -(-cols // 128)
    full = torch.zeros(nr * step, nc * 128, dtype=torch.float64)
    full[:rows, :cols] = x
    tiles = full.view(nr, step, nc, 128)
    bad = ~torch.isfinite(tiles).all(3).all(1)
    amax = torch.where(torch.isfinite(tiles), tiles.abs(), torch.zeros_like(tiles)).amax((1, 3))
    e = torch.zeros(nr, nc, dtype=torch.int64)
    # the least e >= -127 with amax <= 448 * 2^e, tried out: no logarithm to be off by one
    e[:] = -127
    for _ in range(260):
        e += (amax > 448.0 * torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double())).long()
    e[amax == 0] = 0
    y = tiles * torch.pow(torch.tensor(2.0, dtype=torch.float64), -e.double())[:, None, :, None]
    # nearest e4m3, ties to even, from the list of all its values
    codes = torch.arange(0, 127, dtype=torch.uint8)
    vals = codes.view(E4M3).double()
    mag = torch.where(torch.isfinite(y), y.abs(), torch.zeros_like(y)).reshape(-1)
    hi = torch.searchsorted(vals, mag).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dh, dl = vals[hi] - mag, mag - vals[lo]
    pick = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    sign = torch.signbit(y).reshape(-1).to(torch.uint8) * 128
    q = (pick.to(torch.uint8) + sign).view(nr, step, nc, 128)
    q = torch.where(bad[:, None, :, None], torch.full_like(q, 0x7F), q).reshape(nr * step, nc * 128)[:rows, :cols]
    s = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    return q.contiguous(), s.t().contiguous()


def values(q, s):
    """code * scale in 64 bits; q uint8 or e4m3 codes, s uint8 or e8m0 bytes."""
    q, s = q.detach().cpu(), s.detach().cpu()
    v = (q if q.dtype == E4M3 else q.view(E4M3)).double()
    b = (s if s.dtype == torch.uint8 else s.view(torch.uint8))
    f = torch.pow(torch.tensor(2.0, dtype=torch.float64), b.double() - 127)
    f = torch.where(b == 255, torch.full_like(f, float("nan")), f)
    rows, cols = v.shape
    at_r = torch.arange(rows) if f.shape[1] == rows else torch.arange(rows) // 128
    return v * f[(torch.arange(cols) // 128)[None, :], at_r[:, None]]


def spread_bytes(s, rows, cols):
    """Scale bytes as a value per element."""
    s = s.cpu() if s.dtype == torch.uint8 else s.cpu().view(torch.uint8)
    at_r = torch.arange(rows) if s.shape[1] == rows else torch.arange(rows) // 128
    return s[(torch.arange(cols) // 128)[None, :], at_r[:, None]]


def bytes_of(t):
    return t.detach().contiguous().cpu().view(torch.uint8)
