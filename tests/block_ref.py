"""The block-of-128 operators' definitions in 64 bits, with plain torch."""
import torch

BLOCK = 128


def scale_of(amax):
    """Smallest power of two s >= 2^-126 with amax <= 448 s; NaN in amax must have been left out."""
    m, e = torch.frexp(amax.double())  # amax = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(amax == 0, torch.full_like(e, -126), e - 9 + (m > 0.875).to(e.dtype))
    e = torch.where(torch.isinf(amax), torch.full_like(e, 120), e)
    return torch.ldexp(torch.ones_like(m), e.clamp(min=-126))


def e4m3(v):
    """The nearest E4M3 value, ties to even, beyond 448 saturated."""
    mag = v.abs().clamp(max=448.0)
    step = torch.ldexp(torch.ones_like(v), torch.frexp(mag.clamp(min=2.0 ** -6))[1] - 4)
    return torch.copysign(torch.where(torch.isnan(v), v, torch.round(mag / step) * step), v)


def amax_skip_nan(v, dims):
    return torch.nan_to_num(v.abs(), nan=0.0, posinf=float("inf")).amax(dims)


def _blocked(v, dim):
    n = v.size(dim)
    pad = (-n) % BLOCK
    if pad:
        shape = list(v.shape)
        shape[dim] = pad
        v = torch.cat([v, v.new_zeros(shape)], dim)
    return v.unflatten(dim, (-1, BLOCK))


def rows(x):
    """(values (T, C), scale (C / 128, T)) of blocks along rows; both 64 bits."""
    b = _blocked(x.double(), 1)
    s = scale_of(amax_skip_nan(b, 2))
    return e4m3(b / s[..., None]).flatten(1)[:, :x.size(1)], s.t()


def weight(w):
    """(values, scale) of blocks of 128 x 128 of a (n, k) matrix."""
    b = _blocked(_blocked(w.double(), 1), 0)  # (n / 128, 128, k / 128, 128)
    s = scale_of(amax_skip_nan(b, (1, 3)))
    return e4m3(b / s[:, None, :, None]).flatten(2).flatten(0, 1)[:w.size(0), :w.size(1)], s


def tokens(x):
    """What a (T, C) matrix stands for in blocks of 128 rows of a column, and the blocks' scales."""
    b = _blocked(x.double(), 0)
    s = scale_of(amax_skip_nan(b, 1))
    return (e4m3(b / s[:, None]) * s[:, None]).flatten(0, 1)[:x.size(0)], s


def row_values(x):
    v, s = rows(x)
    return v * s.t().repeat_interleave(BLOCK, 1)[:, :x.size(1)]


def weight_values(data, scale):
    n, k = data.shape
    return data.double() * scale.double().repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def spans(ends, rows_):
    """[(first, last)] of the experts, ends held to what they may be."""
    out, before = [], 0
    for e in ends:
        e = max(min(max(int(e), 0), rows_), before)
        out.append((before, e))
        before = e
    return out


def product_bound(k, magnitude):
    """How far an fp32 sum over k products may be from the exact one where the products' magnitudes add up to `magnitude`: every
    product is exact in fp32 or finer; each of k / 32 MMAs adds 33 numbers, each of k / 128 blocks is scaled and added. An adder
    may cut instead of round: one unit of 2^-23 of the running sum each."""
    return (k / 32 + 33 + 3 * (k / 128 + 1)) * 2.0 ** -23 * magnitude
