"""Microscaled blocks in 64 bits, written from their definition: the references of the tests."""
import torch

GRID4 = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def scale_bytes(x, emax):
    """x [..., K] to scale bytes [..., K/32]: the exponent of the largest magnitude minus emax, biased
    by 127, not below 0; 255 where a block holds an infinity or a NaN."""
    b = x.double().unflatten(-1, (-1, 32)).abs()
    bad = ~torch.isfinite(b).all(-1)
    top = torch.where(torch.isfinite(b), b, torch.zeros_like(b)).amax(-1)
    _, e = torch.frexp(top)  # top = m 2^e, m in [0.5, 1)
    s = torch.where(top > 0, e.double() - 1 - emax + 127, torch.zeros_like(top)).clamp(min=0)
    return torch.where(bad, torch.full_like(s, 255), s).to(torch.uint8)


def _by_block(x, s):
    scale = torch.exp2(s.double() - 127)
    return x.double().unflatten(-1, (-1, 32)), scale.unsqueeze(-1)


def quantize4(x, s=None):
    """(codes 0..15 one a byte [..., K], scale bytes); non-finite blocks have code 0 here."""
    s = scale_bytes(x, 2) if s is None else s
    b, scale = _by_block(x, s)
    v = torch.nan_to_num(b / scale, nan=0.0, posinf=0.0, neginf=0.0)
    a = v.abs().clamp(max=6.0)
    grid = GRID4.to(x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    up_on_tie = (torch.arange(7, device=x.device) % 2 == 1)  # from an odd code up to the even one
    code = ((a.unsqueeze(-1) > mid) | ((a.unsqueeze(-1) == mid) & up_on_tie)).sum(-1)
    code = code + 8 * torch.signbit(b).long()
    return code.flatten(-2).to(torch.uint8), s


def values4(code, s):
    """What codes (one a byte) and scale bytes stand for."""
    v = GRID4.to(code.device)[(code & 7).long()] * (1 - 2 * (code >> 3).double())
    b, scale = _by_block(v, s)
    scale = torch.where(s.unsqueeze(-1) == 255, torch.full_like(scale, float("nan")), scale)
    return (b * scale).flatten(-2)


def held4(x, s=None):
    return values4(*quantize4(x, s))


def held8(x, s=None):
    """x as its 8-bit blocks hold it: e4m3, ties to even, saturating at 448."""
    s = scale_bytes(x, 8) if s is None else s
    b, scale = _by_block(x, s)
    a = (b / scale).abs().clamp(max=448.0)
    _, e = torch.frexp(a)
    step = torch.exp2((e.double() - 1).clamp(min=-6) - 3)
    v = torch.round(a / step) * step * torch.where(torch.signbit(b), -1.0, 1.0)
    v = torch.where(s.unsqueeze(-1) == 255, torch.full_like(v, float("nan")), v * scale)
    return v.flatten(-2)


def unpack4(codes):
    """Packed codes [..., K/2] to one a byte [..., K]."""
    return torch.stack((codes & 15, codes >> 4), -1).flatten(-2)


def pack4(code):
    return (code[..., 0::2] | (code[..., 1::2] << 4)).contiguous()


def tile_order(s, rows_of_tiles=None):
    """Scale bytes [rows][K/32] of one segment to the tiles' order, [tiles][chunks][512] (bytes of
    rows that do not exist are 0 here)."""
    rows, blocks = s.shape
    chunks = (blocks + 7) // 8 * 2
    tiles = (rows + 127) // 128
    full = torch.zeros(tiles * 128, chunks * 4, dtype=torch.uint8, device=s.device)
    full[:rows, :blocks] = s
    # [tile][row/32][row%32][chunk][block] -> [tile][chunk][row%32][row/32][block]
    return full.reshape(tiles, 4, 32, chunks, 4).permute(0, 3, 2, 1, 4).reshape(tiles, chunks, 512).contiguous()


def candidates(x, rel, held, emax):
    """The least and the largest value that x(1 +- rel) may be held as, whatever the errors of the
    block's other values: the scale may be that of the largest magnitude times 1 - rel or 1 + rel."""
    lo = hi = None
    for f in (1 - rel, 1 + rel):
        s = scale_bytes(x * f, emax)
        for g in (1 - rel, 1 + rel):
            v = held(x * g, s)
            lo = v if lo is None else torch.minimum(lo, v)
            hi = v if hi is None else torch.maximum(hi, v)
    return lo, hi


def ffn_backward(x, g, u, d_o, wg, wu, wd):
    """One expert's gradients in 64 bits from the gate's and up projection's outputs as kept:
    (d_x, d_wg, d_wu, d_wd) and the intermediates the error bounds need."""
    s = torch.sigmoid(g)
    d_h = d_o @ wd.T
    slope = s * (1 + g * (1 - s))
    d_g, d_u, h = d_h * u * slope, d_h * g * s, g * s * u
    return (d_g @ wg.T + d_u @ wu.T, x.T @ d_g, x.T @ d_u, h.T @ d_o), (d_h, s, d_g, d_u, h)
