"""The 8-bit functions with block scales in 64 bits, from their definition, and the bounds that their roundings give."""

from __future__ import annotations

import torch

BLOCK = 128
E4M3 = torch.float8_e4m3fn
U24 = 2.0 ** -24  # half a step of fp32, relative


def blocks(n: int) -> int:
    return -(-n // BLOCK)


def nearest(q):
    """The e4m3 values nearest to q (|q| up to 448), ties to even; and half a step there."""
    _, e = torch.frexp(q.abs().clamp(min=2.0 ** -6))
    step = torch.exp2((e - 1).double() - 3)
    return torch.round(q / step) * step, step / 2


def block_max(y, rows):
    """Largest |y| of each block, at least 2^-100; NaN where a block has a NaN or an infinity."""
    m, k = y.shape
    full = torch.zeros(blocks_of(m, rows) * rows, blocks(k) * BLOCK, dtype=torch.float64, device=y.device)
    full[:m, :k] = y
    a = full.view(-1, rows, blocks(k), BLOCK).abs().amax((1, 3))
    return torch.where(a.isfinite(), a.clamp(min=2.0 ** -100), torch.nan)


def blocks_of(m, rows):
    return -(-m // rows)


def spread(scales, rows, m, k):
    """A block's value at each of its places [m, k]."""
    return scales.repeat_interleave(rows, 0)[:m].repeat_interleave(BLOCK, 1)[:, :k]


def rounded(y, rows):
    """(quotients 448 y / a, a / 448) of y [m, k] in blocks of `rows` rows."""
    a = block_max(y, rows)
    return 448 * y / spread(a, rows, *y.shape), a / 448


def check_codes(codes, q, loose=0.0):
    """Codes are those nearest to q, whose own error is at most `loose` relative; NaN where q is."""
    got, want = codes.double(), q
    assert torch.equal(got.isnan(), want.isnan())
    got, want = got.nan_to_num(), want.nan_to_num()
    near, half = nearest(want)
    if loose == 0.0:
        assert torch.equal(got, near)
    else:
        # next to a power of two the step above is the larger one
        _, more = nearest(want.abs() * (1 + 2 * loose))
        off = (got - want).abs() - torch.maximum(half, more) - loose * want.abs()
        assert off.max() <= 0, off.max()


def check_scales(got, want, loose):
    assert got.dtype == torch.float32
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan())
    off = ((got - want).abs() - loose * want.abs()).nan_to_num()
    assert off.max() <= 0, (off / want.abs()).nan_to_num().max()


def product(x, sx, w, sw):
    """(y, the sum of the terms' sizes) of codes x [m, k], scales [m, kb] and w [n, k], [nb, kb] in 64 bits."""
    a = x.double() * spread(sx.double(), 1, *x.shape)
    b = w.double() * spread(sw.double(), BLOCK, *w.shape)
    return a @ b.T.contiguous(), a.abs() @ b.T.abs().contiguous()


def check_product(y, x, sx, w, sw):
    """y against 64 bits.  With S the sum of the terms' sizes: a block's sum of 128 exact products is off by at most
    128 half steps of fp32 (in whatever order; 2 * 128 for an adder that cuts instead of rounding), the two factors'
    product and its product with the sum by 2 more, the sum over the blocks by one for each.

    bf16 results come from the 8-bit matrix instructions, which drop of up to 16 neighbouring products what lies 2^-13
    below the largest one: less than 2^-13 of it for each of the 15 others.  The result is rounded to bf16 by half a step.
    The second bound is one of all values together, where what is dropped (some 2^-16) does not add up."""
    want, size = product(x, sx, w, sw)
    bound = (2 * BLOCK + 4 + sx.shape[1]) * U24 * size
    got = y.double()
    if y.dtype == torch.bfloat16:
        bound = bound + 15 * 2.0 ** -13 * size
        bound = bound + 2.0 ** -8 * (want.abs() + bound) + 2.0 ** -134
        assert (got - want).norm() <= 1.01 * 2.0 ** -8 * want.norm() + 2.0 ** -12 * (size.norm() / size.shape[1] ** 0.5)
    off = (got - want).abs() - bound - 2.0 ** -149
    assert off.max() <= 0, (off.max(), ((got - want).abs() / size.clamp(min=1e-300)).max())
