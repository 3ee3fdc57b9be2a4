"""The 8-bit functions with block scales on the GPU against their definition in 64 bits: codes of bf16 values exactly,
sums within the bound that their roundings give, and the functions together as a layer uses them."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from triton_kernels import _hip
    from triton_kernels import fp8_blocks as F

import fp8_blocks_ref as R
import test_fp8_blocks_cpu as C

DEV = "cuda"
BF, F32, E4 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
U24 = R.U24


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rnd(*shape, seed=0, dtype=BF, std=1.0):
    return (torch.randn(*shape, generator=gen(seed), device=DEV) * std).to(dtype)


def strided(t, gap=8, fill=math.nan, before=0):
    """t's values as a view of rows `gap` further apart, `before` values into a buffer of `fill`."""
    *lead, n, k = t.shape
    buf = torch.full((math.prod(lead) * n * (k + gap) + before,), fill, device=DEV).to(t.dtype)
    view = buf[before:].view(*lead, n, k + gap)[..., :k]
    view.copy_(t)
    return view


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------- rounding
# a bf16 value times 7/8 and the quotient are exact where the quotient is a code or half way between two; fp32 values are
# rounded once before the quotient's rounding: two half steps
LOOSE = {BF: 0.0, F32: 2 * U24}
SHAPES = [(1, 1), (1, 127), (1, 128), (1, 129), (2, 8), (3, 200), (5, 136), (16, 2048), (17, 1408), (33, 2050), (64, 10944),
          (700, 260), (4099, 64), (33001, 264), (9001, 1411)]  # the last: two blocks a lane
LARGE = [(70003, 1408), (130001, 136)]  # past the last-level cache


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,k", SHAPES)
def test_rows_are_rounded_to_the_nearest_codes(m, k, dtype):
    x = rnd(m, k, seed=m + k, dtype=dtype) * torch.exp(2 * rnd(m, 1, seed=k, dtype=F32)).to(dtype)
    for v in (x, strided(x), strided(x, gap=3, before=1)):
        codes, scales = F.quantize_fp8_blocks(v)
        q, s = R.rounded(x.double(), 1)
        R.check_codes(codes, q, LOOSE[dtype])
        R.check_scales(scales, s, U24)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [(1, 1), (127, 128), (128, 128), (129, 136), (300, 200), (257, 2050), (2, 130, 136), (3, 70, 65),
                                   (64, 16, 24)])
def test_weights_are_rounded_in_blocks_of_128_rows(shape, dtype):
    x = rnd(*shape, seed=sum(shape), dtype=dtype)
    for v in (x, strided(x), strided(x, gap=3, before=1)):
        codes, scales = F.quantize_fp8_blocks(v, 128)
        for c, s, w in zip(codes.view(-1, *shape[-2:]), scales.view(-1, *scales.shape[-2:]), x.view(-1, *shape[-2:])):
            q, want = R.rounded(w.double(), 128)
            R.check_codes(c, q, LOOSE[dtype])
            R.check_scales(s, want, U24)


def test_every_bf16_value_against_every_kind_of_largest():
    """All finite bf16 values below a largest one, for largest ones of all mantissas and the ends of the range: ties too."""
    bits = torch.arange(0x7f80, dtype=torch.int32, device=DEV).to(torch.int16).view(BF)
    tops = [0x3f80 + i for i in range(128)] + [0x0080, 0x0d80, 0x0d7f, 0x0d00, 0x2000, 0x7f7f, 0x7f00]
    for top in tops:
        a = torch.tensor([top], dtype=torch.int16, device=DEV).view(BF)
        v = bits[:top + 1]
        v = torch.cat([v, -v])
        n = -(-v.numel() // 127) * 127
        v = torch.cat([v, v.new_zeros(n - v.numel())]).view(-1, 127)
        x = torch.cat([v, a.expand(v.shape[0], 1)], 1).contiguous()
        codes, scales = F.quantize_fp8_blocks(x)
        q, s = R.rounded(x.double(), 1)
        R.check_codes(codes, q)
        R.check_scales(scales, s, U24)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_blocks_of_zeros_and_of_values_that_are_none(dtype):
    x = rnd(6, 300, seed=1, dtype=dtype)
    x[0] = 0
    x[1, 128:256] = 0
    x[2, 5] = math.nan
    x[3, 200] = math.inf
    x[4, 299] = -math.inf
    x[5, :128] = 2.0 ** -120
    x[5, 130] = 2.0 ** 127
    codes, scales = F.quantize_fp8_blocks(x)
    q, s = R.rounded(torch.where(x.isfinite(), x, math.nan).double(), 1)
    for r, b in ((2, 0), (3, 1), (4, 2)):
        q[r, 128 * b:128 * b + 128] = math.nan
    R.check_codes(codes, q, LOOSE[dtype])
    R.check_scales(scales, s, U24)
    codes, scales = F.quantize_fp8_blocks(x, 128)
    assert codes[:, :256].isnan().all() and codes[:, 256:].isnan().all() and scales.isnan().all()
    assert F.quantize_fp8_blocks(x.new_zeros(130, 130), 128)[0].float().count_nonzero() == 0


@pytest.mark.parametrize("m", [1, 3, 1024, 1025, 1200])
@pytest.mark.parametrize("k", [1, 64, 200, 512, 513, 1030, 2048, 2049, 5120, 8192, 8200, 10944])
@pytest.mark.parametrize("dtype,residual", [(BF, True), (BF, False), (F32, True), (F32, False)])
def test_norm(m, k, dtype, residual):
    if m > 3 and k > 2049:
        m = m // 8
    x, r = rnd(m, k, seed=m + k, dtype=dtype, std=3), rnd(m, k, seed=m * k, dtype=dtype)
    w = (1 + 0.3 * rnd(k, seed=k, dtype=F32)).to(dtype)
    h = (x.float() + r.float()).to(dtype) if residual else x
    hd = h.double()
    q, s = R.rounded(hd * w.double(), 1)
    s = s / torch.sqrt((hd * hd).mean(1, keepdim=True) + 1e-6)
    # the sum of squares: a lane adds up to ceil(k / 512) * 8 of them one after another, then eight partial sums
    # meet; half of that, and eight roundings of the factor and the scale
    loose = (-(-k // 512) * 4 + 4 + 8) * U24
    for v in (0, 1, 2):
        a = (x, strided(x, 16), strided(x, 5, before=1))[v]
        b = (r, strided(r, 8), strided(r, 3, before=3))[v]
        out = F.rmsnorm_fp8_blocks(a, w, 1e-6, b if residual else None)
        # fp32: the product h w is rounded, then as the rows
        R.check_codes(out[0], q, LOOSE[dtype] + (U24 * 2 if dtype == F32 else 0))
        R.check_scales(out[1], s, loose)
        assert len(out) == 2 + residual
        if residual:
            assert torch.equal(out[2], h)


def test_norm_of_rows_of_zeros_and_with_values_that_are_none():
    for dtype in (BF, F32):
        x = rnd(5, 300, seed=2, dtype=dtype)
        x[0] = 0
        x[1, 250] = math.nan
        x[2, 3] = math.inf
        w = torch.ones(300, device=DEV, dtype=dtype)
        codes, scales, h = F.rmsnorm_fp8_blocks(x, w, 1e-6, torch.zeros_like(x))
        assert not codes[0].float().any() and scales[0].isfinite().all()
        # the row's factor is NaN, or with an infinity 0: what the scales stand for is not finite in the block that has it
        assert scales[1].isnan().all()
        assert codes[2, :128].isnan().all() and scales[2, 0].isnan()
        assert codes[3:].float().isfinite().all() and scales[3:].isfinite().all()
        # what rows do not hold is not read
        assert torch.equal(F.rmsnorm_fp8_blocks(x[3:], w, 1e-6)[0].view(torch.uint8), codes[3:].view(torch.uint8))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,k", SHAPES)
def test_silu_mul(m, k, dtype):
    both = rnd(m, 2 * k, seed=m + k, dtype=dtype, std=4)
    both[:, ::7] *= 5  # gates down to -80
    for gate, up in (both.chunk(2, 1), (strided(both, 1, before=1)[:, :k], both[:, k:])):
        codes, scales = F.silu_mul_fp8_blocks(gate, up)
        y = gate.double() * torch.sigmoid(gate.double()) * up.double()
        q, s = R.rounded(y, 1)
        # exp to an ulp, its correction, the sum, the quotient, two products: 8 half steps; both values of a quotient
        R.check_codes(codes, q, 2 * 8 * U24 + 3 * U24)
        R.check_scales(scales, s, 9 * U24)


@pytest.mark.parametrize("m,k", LARGE)
def test_rows_past_the_last_level_cache(m, k):
    both = rnd(m, 2 * k, seed=k, dtype=F32 if k < 200 else BF, std=2)
    if k < 200:
        both = strided(both, 1030)[:, :2 * k]  # far apart: 1.3 GB between the first and the last
    gate, up = both.chunk(2, 1)
    for codes, scales, y, loose in ((*F.silu_mul_fp8_blocks(gate, up), gate.double() * torch.sigmoid(gate.double()) * up, 19 * U24),
                                    (*F.quantize_fp8_blocks(both), both.double(), LOOSE[both.dtype])):
        q, s = R.rounded(y.double(), 1)
        R.check_codes(codes, q, loose)
        R.check_scales(scales, s, 9 * U24)


def test_silu_mul_at_the_ends():
    g = torch.tensor([0.0, -0.0, 80.0, -80.0, 88.0, -88.0, 100.0, -83.2, -84.0, 1e30, -1e30, 1e-30, -87.5], device=DEV)
    u = torch.full_like(g, 2.0)
    for i in range(len(g)):
        gi, ui = g[i:i + 1].view(1, 1), u[i:i + 1].view(1, 1)
        codes, scales = F.silu_mul_fp8_blocks(gi, ui)
        want = (gi.double() * torch.sigmoid(gi.double()) * ui.double()).item()
        got = (codes.double() * scales.double()).item()
        assert abs(got - want) <= 2.0 ** -20 * abs(want) + 2.0 ** -110, (g[i], got, want)
    for bad in (math.nan, math.inf, -math.inf):
        for pair in ((bad, 1.0), (1.0, bad)):
            x = torch.ones(2, 2, 256, device=DEV)
            x[0, 0, 3], x[1, 0, 3] = pair
            codes, scales = F.silu_mul_fp8_blocks(x[0], x[1])
            assert codes[0, :128].isnan().all() and scales[0, 0].isnan()
            assert codes[0, 128:].float().isfinite().all() and scales[0, 1].isfinite() and scales[1].isfinite().all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_silu_mul_where_the_exponential_is_no_normal_number(dtype):
    """Gates down to -3e38, with factors that bring the product back to codes: blocks of one value and of 128."""
    g = torch.cat([torch.arange(-200, -80, 0.25), torch.tensor([-250.0, -1000.0, -1e30, -3e38, -3.3e38])])
    u = 2.0 ** torch.arange(0, 128, 3.0)
    gate, up = (v.reshape(-1, 1).to(DEV, dtype) for v in torch.meshgrid(g, u, indexing="ij"))
    for cols in (1, 128):
        n = gate.numel() // cols * cols
        a, b = gate[:n].view(-1, cols), up[:n].view(-1, cols)
        codes, scales = F.silu_mul_fp8_blocks(a, b)
        q, s = R.rounded(a.double() * torch.sigmoid(a.double()) * b.double(), 1)
        R.check_codes(codes, q, 2 * 8 * U24 + 3 * U24)
        R.check_scales(scales, s, 9 * U24)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_silu_mul_of_gates_up_to_the_largest(dtype):
    """Gates up to the type's largest, with factors that leave their product in range: blocks of one value and of 128."""
    g = torch.cat([torch.tensor([60.0, 88.0, 90.0, 104.0, 128.0, 1e4, 1e20, 2.3e38, 2.35e38, 2.36e38, 2.4e38, 3e38, 3.3e38]),
                   torch.tensor([torch.finfo(dtype).max])])
    u = torch.cat([s * 2.0 ** -torch.arange(0, 127, 3.0) for s in (1.0, -1.0)])
    gate, up = (v.reshape(-1, 1).to(DEV, dtype) for v in torch.meshgrid(g, u, indexing="ij"))
    assert gate.isfinite().all()
    for cols in (1, 128):
        n = gate.numel() // cols * cols
        a, b = gate[:n].view(-1, cols), up[:n].view(-1, cols)
        codes, scales = F.silu_mul_fp8_blocks(a, b)
        q, s = R.rounded(a.double() * torch.sigmoid(a.double()) * b.double(), 1)
        R.check_codes(codes, q, 2 * 8 * U24 + 3 * U24)
        R.check_scales(scales, s, 9 * U24)


def test_silu_mul_rounds_the_quotient_once():
    """Blocks of one value, up = 1: the scale is silu(g) / 448.  1 + exp(-g) is rounded by up to half a step of numbers
    from 1 to 2 and holds exp(-g) to 8 half steps; then the quotient's rounding and the scale's, half a step of each."""
    gate = torch.linspace(8, 12, 2 ** 20, dtype=torch.float64, device=DEV).float().view(-1, 1)
    codes, scales = F.silu_mul_fp8_blocks(gate, torch.ones_like(gate))
    assert (codes.float() == 448).all()
    e = torch.exp(-gate.double())
    y = gate.double() / (1 + e)

    def half(v):  # half a step at v, relative; of the larger step where v is next to a power of two
        return torch.exp2(torch.floor(torch.log2(v * (1 + 2.0 ** -20)))) * U24 / v

    bound = (U24 / (1 + e) + 8 * U24 * e + half(y) + half(y / 448)) * (1 + 2.0 ** -20)
    off = (scales.double() * 448 / y - 1).abs()
    assert (off <= bound).all(), (off / bound).max()


# ---------------------------------------------------------------- products
def matrix(n, k, seed, rows, groups=None):
    x = rnd(*(() if groups is None else (groups,)), n, k, seed=seed, dtype=F32)
    x = x * torch.exp(rnd(*x.shape[:-1], 1, seed=seed + 1, dtype=F32))
    return F.quantize_fp8_blocks(x, rows)


def guarded(codes, scales, gap, before):
    """Codes and scales as views between NaNs."""
    *lead, n, k = codes.shape
    buf = torch.full((math.prod(lead) * n * (k + gap) + before + 64,), 0x7f, dtype=torch.uint8, device=DEV)
    c = buf[before:before + math.prod(lead) * n * (k + gap)].view(*lead, n, k + gap)[..., :k]
    c.copy_(codes.view(torch.uint8))
    return c.view(E4), strided(scales, 3)


MS = [1, 2, 15, 16, 17, 33, 64, 65, 129, 300]
NK = [(1, 1), (16, 128), (17, 127), (130, 129), (64, 16), (300, 144), (100, 2048), (3648, 2048), (257, 1408), (50, 10944),
      (1000, 2000), (129, 4099)]


@pytest.mark.parametrize("n,k", NK)
@pytest.mark.parametrize("m", MS)
def test_linear(m, n, k):
    x, sx = matrix(m, k, m + k, 1)
    w, sw = matrix(n, k, n * k, 128)
    for dtype in (BF, F32):
        R.check_product(F.linear_fp8_blocks(x, sx, w, sw, dtype), x, sx, w, sw)
    for gap, before in ((16, 0), (5, 3)):
        got = F.linear_fp8_blocks(*guarded(x, sx, gap, before), *guarded(w, sw, gap, before), F32)
        R.check_product(got, x, sx, w, sw)


@pytest.mark.parametrize("m,n,k", [(1025, 2816, 2048), (2048, 2050, 1408), (4099, 300, 656), (513, 10944, 256), (700, 21888, 128),
                                   (3000, 3000, 300)])
def test_linear_large(m, n, k):
    x, sx = matrix(m, k, m + k, 1)
    w, sw = matrix(n, k, n * k, 128)
    for dtype in (BF, F32):
        R.check_product(F.linear_fp8_blocks(x, sx, w, sw, dtype), x, sx, w, sw)


@pytest.mark.parametrize("m", [1, 20, 100, 600])
def test_linear_sums_whole_numbers_exactly(m):
    """Codes that are small whole numbers and scales that are powers of two: every sum is exact in fp32, so each row
    has to meet each weight and each block its own two scales, without a tolerance."""
    g = gen(m)
    n, k = 515, 1200
    x = torch.randint(-4, 5, (m, k), device=DEV, generator=g).float()
    w = torch.randint(-4, 5, (n, k), device=DEV, generator=g).float()
    sx = torch.exp2(torch.randint(-2, 3, (m, R.blocks(k)), device=DEV, generator=g).float())
    sw = torch.exp2(torch.randint(-2, 3, (R.blocks(n), R.blocks(k)), device=DEV, generator=g).float())
    got = F.linear_fp8_blocks(x.to(E4), sx, w.to(E4), sw, F32)
    want, _ = R.product(x.to(E4), sx, w.to(E4), sw)
    assert torch.equal(got.double(), want)
    assert torch.equal(F.linear_fp8_blocks(x.to(E4), sx, w.to(E4), sw), want.to(BF))


@pytest.mark.parametrize("m", [1, 40, 600])
def test_linear_whose_largest_terms_cancel(m):
    """Two terms of 448 * 448 and opposite sign, the others multiples of 2^-6 up to 1: what is left after them is exact in
    fp32 results, whose every partial sum has 24 bits.  bf16 results may lose 15 * 2^-13 of each of the two."""
    g = gen(m)
    n, k = 150, 300
    small = lambda rows: torch.randint(-8, 9, (rows, k), device=DEV, generator=g) / 8
    sx, sw = torch.ones(m, R.blocks(k), device=DEV), torch.ones(R.blocks(n), R.blocks(k), device=DEV)
    for a, b in ((0, 1), (3, 18), (5, 69), (0, 127), (200, 299), (100, 140)):
        x, w = small(m), small(n)
        x[:, a] = x[:, b] = w[:, a] = 448
        w[:, b] = -448
        x, w = x.to(E4), w.to(E4)
        want, size = R.product(x, sx, w, sw)
        assert torch.equal(F.linear_fp8_blocks(x, sx, w, sw, F32).double(), want)
        off = (F.linear_fp8_blocks(x, sx, w, sw).double() - want).abs()
        assert (off <= 15 * 2.0 ** -13 * size + 2.0 ** -8 * want.abs() * 1.01).all()


def test_linear_of_every_code_and_of_none():
    """The 254 finite codes times one, NaN codes, infinite and NaN scales."""
    codes = torch.arange(256, dtype=torch.uint8, device=DEV).view(256, 1).view(E4)
    one, s1 = torch.ones(1, 1, device=DEV).to(E4), torch.ones(1, 1, device=DEV)
    sx = torch.ones(256, 1, device=DEV)
    got = F.linear_fp8_blocks(codes, sx, one, s1, F32)[:, 0]
    want = codes.view(256).float()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    x, xs = matrix(40, 300, 3, 1)
    w, ws = matrix(200, 300, 4, 128)
    clean = F.linear_fp8_blocks(x, xs, w, ws)
    xs[3, 1] = math.nan
    xs[7, 2] = math.inf
    ws[1, 0] = math.nan
    got = F.linear_fp8_blocks(x, xs, w, ws)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[3], bad[7], bad[:, 128:] = True, True, True
    assert not got[bad].isfinite().any() and got[3].isnan().all() and got[:, 128:].isnan().all()
    assert torch.equal(got[~bad], clean[~bad])


def test_products_leave_what_is_not_theirs():
    """Through the C ABI with rows of y further apart than N: the gaps and the rows of no group stay."""
    x, sx = matrix(70, 300, 5, 1)
    w, sw = matrix(130, 300, 6, 128, groups=3)
    for dtype, code in ((BF, 0), (F32, 1)):
        for ys, at in ((136, 0), (131, 1)):
            buf = torch.full((70 * ys + 9,), 7.0, device=DEV).to(dtype)
            y = buf[at:at + 70 * ys].view(70, ys)
            _hip.call("dsv2_linear_fp8_blocks", x.data_ptr(), 300, sx.data_ptr(), 3, 70, 300, w.data_ptr(), 300,
                      sw.data_ptr(), 3, 130, y.data_ptr(), ys, code, _hip.stream_ptr())
            R.check_product(y[:, :130], x, sx, w[0], sw[0])
            assert (y[:, 130:] == 7).all() and (buf[:at] == 7).all() and (buf[at + 70 * ys:] == 7).all()
            buf.fill_(7.0)
            offsets = i32([4, 20, 20, 66])
            _hip.call("dsv2_grouped_linear_fp8_blocks", x.data_ptr(), 300, sx.data_ptr(), 3, 70, None, 70, 300, w.data_ptr(),
                      130 * 300, 300, sw.data_ptr(), 6, 3, 130, 3, offsets.data_ptr(), y.data_ptr(), ys, code,
                      _hip.stream_ptr())
            for e, (lo, hi) in ((0, (4, 20)), (2, (20, 66))):
                R.check_product(y[lo:hi, :130], x[lo:hi], sx[lo:hi], w[e], sw[e])
            assert (y[:4] == 7).all() and (y[66:] == 7).all() and (y[:, 130:] == 7).all()


@pytest.mark.parametrize("inter", [200, 203, 256])
def test_gate_and_up_with_scales_of_their_own_into_one_buffer(inter):
    """Through the C ABI: halves that are no whole blocks of 128 rows, as two products with the row stride of both; whole
    blocks one behind the other, as one."""
    r, h, kb, ib = 33, 300, 3, R.blocks(inter)
    x, sx = matrix(r, h, 5, 1)
    gate, up = matrix(inter, h, 6, 128), matrix(inter, h, 7, 128)
    y = torch.zeros(r, 2 * inter, device=DEV, dtype=BF)
    for (w, sw), at in ((gate, 0), (up, inter)):
        _hip.call("dsv2_linear_fp8_blocks", x.data_ptr(), h, sx.data_ptr(), kb, r, h, w.data_ptr(), h, sw.data_ptr(), kb,
                  inter, y.data_ptr() + 2 * at, 2 * inter, 0, _hip.stream_ptr())
    for (w, sw), half in zip((gate, up), y.chunk(2, 1)):
        R.check_product(half, x, sx, w, sw)
    if inter % 128 == 0:
        w = torch.cat([gate[0].view(torch.uint8), up[0].view(torch.uint8)]).view(E4)
        assert torch.equal(F.linear_fp8_blocks(x, sx, w, torch.cat([gate[1], up[1]])), y)
    codes = torch.empty(r, inter, device=DEV, dtype=E4)
    scales = torch.empty(r, ib, device=DEV)
    _hip.call("dsv2_silu_mul_fp8_blocks", y.data_ptr(), 2 * inter, y.data_ptr() + 2 * inter, 2 * inter, r, inter, 0,
              codes.data_ptr(), scales.data_ptr(), _hip.stream_ptr())
    g, u = y.double().chunk(2, 1)
    q, s = R.rounded(g * torch.sigmoid(g) * u, 1)
    R.check_codes(codes, q, 19 * U24)
    R.check_scales(scales, s, 9 * U24)


def check_grouped(y, x, sx, w, sw, offsets, rows=None):
    for e, (lo, hi) in enumerate(zip(offsets, offsets[1:])):
        if hi > lo:
            at = torch.arange(lo, hi, device=DEV) if rows is None else rows[lo:hi].long()
            there = (at >= 0) & (at < x.shape[0])
            at = at.clamp(0, max(x.shape[0] - 1, 0))
            xe = x.view(torch.uint8)[at].view(E4)
            R.check_product(y[lo:hi], xe, torch.where(there[:, None], sx[at], 0), w[e], sw[e])


def offsets_of(counts):
    return [sum(counts[:i]) for i in range(len(counts) + 1)]


@pytest.mark.parametrize("n,k", [(130, 300), (64, 128), (2816, 2048), (257, 1413), (1, 1)])
@pytest.mark.parametrize("counts", [[1], [0, 1], [5, 0, 70, 1, 0], [0] * 70 + [3] + [0] * 60 + [65], [1] * 64, [16] * 20,
                                    [300, 2, 129, 64], [0, 0, 700]], ids=str)
def test_grouped(counts, n, k):
    if n == 2816:
        counts = counts[-5:]
    offsets, groups = offsets_of(counts), len(counts)
    total, tokens = offsets[-1], max(1, offsets[-1] // 3)
    w, sw = matrix(n, k, n + k, 128, groups)
    x, sx = matrix(total, k, total, 1)
    for dtype in (BF, F32):
        check_grouped(F.grouped_linear_fp8_blocks(x, sx, w, sw, i32(offsets), None, dtype), x, sx, w, sw, offsets)
    rows = torch.randint(0, tokens, (total,), generator=gen(k), device=DEV).int()
    x, sx = matrix(tokens, k, total, 1)
    check_grouped(F.grouped_linear_fp8_blocks(x, sx, w, sw, i32(offsets), rows, F32), x, sx, w, sw, offsets, rows)
    for gap, before in ((16, 0), (5, 3)):
        got = F.grouped_linear_fp8_blocks(*guarded(x, sx, gap, before), *guarded(w, sw, gap, before), i32(offsets), rows)
        check_grouped(got, x, sx, w, sw, offsets, rows)


@pytest.mark.parametrize("counts", [[700, 3000, 0, 1500, 12, 1700], [1100] * 8])
def test_grouped_large(counts):
    offsets = offsets_of(counts)
    for n, k, gather in ((2816, 2048, True), (2048, 1408, False), (700, 300, True)):
        w, sw = matrix(n, k, n + k, 128, len(counts))
        tokens = 1500 if gather else offsets[-1]
        x, sx = matrix(tokens, k, 1, 1)
        rows = torch.randint(0, tokens, (offsets[-1],), generator=gen(k), device=DEV).int() if gather else None
        check_grouped(F.grouped_linear_fp8_blocks(x, sx, w, sw, i32(offsets), rows), x, sx, w, sw, offsets, rows)


def rows_for(shape, n, k, groups, f32):
    """The fewest rows of a list with which a product takes that kernel, or None."""
    for m in (1, 11, 20, 48, 100, 130, 256, 300, 520, 700, 1030, 2100, 4100, 9000):
        if _hip.lib.dsv2_linear_fp8_blocks_tiles(m, k, n, groups, int(f32)) == shape:
            return m
    return None


# kernel (dsv2_linear_fp8_blocks_tiles): features with which it is taken, dense and of eight groups
KERNELS = {0: (331, 331), 1: (2809, 201), 2: (8191, 1003), 3: (9003, 20003), 4: (16381, 1003), 5: (16384, 1003), 6: (16384, 2811),
           7: (16381, 8189), 8: (16381, 8187), 10: (65536, 65536), 11: (300, 300), 13: (8191, 1003), 15: (16381, 6001),
           17: (16381, 2811)}
CASES = [(s, g, k) for s, (dense, of8) in KERNELS.items() for g, n in ((0, dense), (8, of8)) if n
         for k in ((1040, 1104, 2064) if s == 1 else (144, 272, 1040, 1104, 2064) if s < 9 else (1040, 2064) if s == 10 else (135, 1041, 1288))]


@pytest.mark.parametrize("shape,groups,k", CASES)
def test_every_kernel(shape, groups, k):
    """Each at lengths that end within a block, between NaNs, results of both types where it gives them."""
    n = KERNELS[shape][groups > 0]
    ran = 0
    for f32 in (False, True):
        m = rows_for(shape, n, k, groups, f32)
        if m is None:
            continue
        ran += 1
        dtype = F32 if f32 else BF
        w, sw = matrix(n, k, n + k, 128, groups or None)
        if shape >= 11:
            gw, gsw = w, sw
        else:
            gw, gsw = guarded(w, sw, 16, 0)
        if not groups:
            x, sx = matrix(m, k, m + k, 1)
            gx, gsx = (x, sx) if shape >= 11 else guarded(x, sx, 16, 0)
            R.check_product(F.linear_fp8_blocks(gx, gsx, gw, gsw, dtype), x, sx, w, sw)
            continue
        cuts = torch.randint(0, m + 1, (groups - 1,), generator=gen(k), device=DEV).sort().values.tolist()
        cuts[2] = cuts[1]  # a group without rows
        offsets = [0, *cuts, m]
        x, sx = matrix(m, k, m + k, 1)
        gx, gsx = (x, sx) if shape >= 11 else guarded(x, sx, 16, 0)
        check_grouped(F.grouped_linear_fp8_blocks(gx, gsx, gw, gsw, i32(offsets), None, dtype), x, sx, w, sw, offsets)
        rows = torch.randint(-1, m + 1, (m,), generator=gen(m), device=DEV).int()
        sx[m // 2:] = torch.where(torch.rand_like(sx[m // 2:]) < 0.01, 0, sx[m // 2:])
        check_grouped(F.grouped_linear_fp8_blocks(x, sx, gw, gsw, i32(offsets), rows, dtype), x, sx, w, sw, offsets, rows)
    assert ran, "no call reaches it"


@pytest.mark.parametrize("shape,groups", [(s, g) for s in KERNELS for g in (0, 8)])
def test_every_kernel_keeps_nans_to_their_rows_and_features(shape, groups):
    """NaN codes and scales that are no numbers, in any block."""
    n, k = KERNELS[shape][groups > 0], 1041 if shape >= 11 else 2064 if shape == 10 else 1040
    ran = 0
    for f32 in (False, True):
        m = rows_for(shape, n, k, groups, f32)
        if m is None:
            continue
        ran += 1
        dtype = F32 if f32 else BF
        w, sw = matrix(n, k, n + k, 128, groups or None)
        x, sx = matrix(m, k, m + k, 1)
        nx, xbad = with_nans(x, 0, 0.05, 1)
        nw, wbad = with_nans(w, 0, 0.01, 2)
        nsx = sx.clone()
        nsx[m // 2, 3] = math.inf
        nsx[m - 1, R.blocks(k) - 1] = math.nan
        xbad[m // 2], xbad[m - 1] = True, True
        nsw = sw.clone()
        nsw[..., 1, R.blocks(k) - 1] = math.nan
        wbad[..., 128:256] = True
        if groups:
            cuts = torch.randint(0, m + 1, (groups - 1,), generator=gen(k), device=DEV).sort().values.tolist()
            offsets = i32([0, *cuts, m])
            wbad = wbad[torch.searchsorted(offsets[1:].contiguous(), torch.arange(m, device=DEV), right=True)]
            clean = F.grouped_linear_fp8_blocks(x, sx, w, sw, offsets, None, dtype)
            got = F.grouped_linear_fp8_blocks(nx, nsx, nw, nsw, offsets, None, dtype)
        else:
            clean, got = F.linear_fp8_blocks(x, sx, w, sw, dtype), F.linear_fp8_blocks(nx, nsx, nw, nsw, dtype)
        check_nans(torch.where(got.isfinite(), got, math.nan), clean, xbad[:, None] | wbad)
    assert ran, "no call reaches it"


@pytest.mark.parametrize("m,n,k", [(4200, 16376, 272), (700, 33000, 144), (9000, 4104, 1296), (4000, 8200, 2176),
                                   (4000, 8194, 1040), (700, 33003, 272)])
def test_large_tiles_one_after_another(m, n, k):
    """More 256 x 256 tiles than workgroups: the next tile's first blocks are read behind the last of the one before, with
    its scales beside them (2, 3, 11 and 17 blocks: within and past their windows of eight)."""
    assert _hip.lib.dsv2_linear_fp8_blocks_tiles(m, k, n, 0, 0) == 8 and -(-m // 256) * -(-n // 256) > 256
    x, sx = matrix(m, k, m + k, 1)
    w, sw = matrix(n, k, n * k, 128)
    y = F.linear_fp8_blocks(x, sx, w, sw)
    R.check_product(y, x, sx, w, sw)
    for _ in range(3):
        assert torch.equal(F.linear_fp8_blocks(x, sx, w, sw), y)


@pytest.mark.parametrize("groups,n,k", [(8, 8184, 1104), (70, 2048, 272), (3, 16387, 2064)])
def test_large_tiles_of_groups(groups, n, k):
    m = 9000
    assert _hip.lib.dsv2_linear_fp8_blocks_tiles(m, k, n, groups, 0) == 8
    cuts = torch.randint(0, m + 1, (groups - 1,), generator=gen(k), device=DEV).sort().values.tolist()
    offsets = [5, *[max(c, 5) for c in cuts], m - 7]
    w, sw = matrix(n, k, n + k, 128, groups)
    x, sx = matrix(2000, k, 1, 1)
    rows = torch.randint(-3, 2003, (m,), generator=gen(m), device=DEV).int()
    y = F.grouped_linear_fp8_blocks(x, sx, w, sw, i32(offsets), rows)
    check_grouped(y, x, sx, w, sw, offsets, rows)
    again = F.grouped_linear_fp8_blocks(x, sx, w, sw, i32(offsets), rows)
    assert torch.equal(again[5:m - 7], y[5:m - 7])


def with_nans(codes, first, share, seed):
    """The codes with a NaN in some rows (`share` of them), in a column from `first` on; and which rows."""
    *lead, k = codes.shape
    bad = torch.rand(*lead, generator=gen(seed), device=DEV) < share
    at = torch.randint(first, k, lead, generator=gen(seed + 1), device=DEV)
    out = codes.view(torch.uint8).clone()
    here = bad[..., None] & (at[..., None] == torch.arange(k, device=DEV))
    return torch.where(here, torch.full_like(out, 0x7f), out).view(E4), bad


def check_nans(got, clean, bad):
    """NaN where a row of x or of w has one, and nowhere else a bit of another value."""
    assert torch.equal(got.isnan(), bad)
    assert torch.equal(torch.where(bad, 0, got), torch.where(bad, 0, clean))


@pytest.mark.parametrize("m,n,k", [(4200, 16376, 272), (700, 33000, 144), (9000, 4104, 1296), (700, 33003, 272)])
def test_large_tiles_keep_nans_to_their_rows_and_features(m, n, k):
    """The sums of a tile's last instructions are added behind its end: none of them may reach the next tile."""
    assert _hip.lib.dsv2_linear_fp8_blocks_tiles(m, k, n, 0, 0) == 8 and -(-m // 256) * -(-n // 256) > 256
    x, sx = matrix(m, k, m + k, 1)
    w, sw = matrix(n, k, n * k, 128)
    clean = F.linear_fp8_blocks(x, sx, w, sw)
    last = (k - 1) // 128 * 128
    nx, xbad = with_nans(x, last, 0.02, 1)
    nw, wbad = with_nans(w, last, 0.02, 2)
    no = torch.zeros_like
    for a, ab, b, bb in ((nx, xbad, w, no(wbad)), (x, no(xbad), nw, wbad), (nx, xbad, nw, wbad)):
        check_nans(F.linear_fp8_blocks(a, sx, b, sw), clean, ab[:, None] | bb)
    # one tile's last 16 rows of each half alone
    nx = x.view(torch.uint8).clone()
    xbad = no(xbad)
    for at in (112, 240):
        nx[256 + at:256 + at + 16, k - 1] = 0x7f
        xbad[256 + at:256 + at + 16] = True
    check_nans(F.linear_fp8_blocks(nx.view(E4), sx, w, sw), clean, xbad[:, None] | no(wbad))


@pytest.mark.parametrize("groups,n,k", [(8, 8184, 1104), (70, 2048, 272), (3, 16387, 2064)])
def test_large_tiles_of_groups_keep_nans_to_their_rows_and_features(groups, n, k):
    m = 9000
    assert _hip.lib.dsv2_linear_fp8_blocks_tiles(m, k, n, groups, 0) == 8
    cuts = torch.randint(0, m + 1, (groups - 1,), generator=gen(k), device=DEV).sort().values.tolist()
    offsets = i32([0, *cuts, m])
    group = torch.searchsorted(offsets[1:].contiguous(), torch.arange(m, device=DEV), right=True)
    w, sw = matrix(n, k, n + k, 128, groups)
    x, sx = matrix(2000, k, 1, 1)
    rows = torch.randint(0, 2000, (m,), generator=gen(m), device=DEV).int()
    clean = F.grouped_linear_fp8_blocks(x, sx, w, sw, offsets, rows)
    last = (k - 1) // 128 * 128
    nx, xbad = with_nans(x, last, 0.02, 1)
    nw, wbad = with_nans(w, last, 0.02, 2)
    xbad = xbad[rows.long()]
    no = torch.zeros_like
    for a, ab, b, bb in ((nx, xbad, w, no(wbad)), (x, no(xbad), nw, wbad), (nx, xbad, nw, wbad)):
        check_nans(F.grouped_linear_fp8_blocks(a, sx, b, sw, offsets, rows), clean, ab[:, None] | bb[group])


@pytest.mark.parametrize("k", [300, 304, 512])
def test_grouped_holds_offsets_and_row_numbers_to_their_ranges(k):
    w, sw = matrix(70, k, 1, 128, 4)
    x, sx = matrix(50, k, 2, 1)
    for given, taken in [([0, 30, 10, 20, 50], [0, 30, 30, 30, 50]), ([-5, 9, 2 ** 31 - 1, 60, 3], [0, 9, 50, 50, 50]),
                         ([50, 40, 30, 20, 10], [50, 50, 50, 50, 50]), ([-2 ** 31, -1, 5, 5, 5], [0, 0, 5, 5, 5])]:
        check_grouped(F.grouped_linear_fp8_blocks(x, sx, w, sw, i32(given), None, F32), x, sx, w, sw, taken)
    rows = torch.arange(50, device=DEV).int()
    rows[::3] = -1
    rows[1::6] = 50
    rows[5], rows[8] = 2 ** 31 - 1, -2 ** 31
    sx[0] = math.nan  # nor does the first row stand in for one that there is not
    rows[rows == 0] = 1
    got = F.grouped_linear_fp8_blocks(x, sx, w, sw, i32([0, 10, 10, 33, 50]), rows, F32)
    check_grouped(got, x, torch.where(sx.isnan(), 0, sx), w, sw, [0, 10, 10, 33, 50], rows)
    assert not got[::3].any()
    none, nosx = F.quantize_fp8_blocks(torch.zeros(0, k, device=DEV))
    assert not F.grouped_linear_fp8_blocks(none, nosx, w, sw, i32([0, 10, 10, 33, 50]), rows).any()


@pytest.mark.parametrize("groups", [130, 4096])
def test_grouped_with_many_groups(groups):
    counts = [(i * 7) % 5 if i % 3 == 0 else 0 for i in range(groups)]
    offsets = offsets_of(counts)
    w, sw = matrix(24, 136, 1, 128, groups)
    x, sx = matrix(offsets[-1], 136, 2, 1)
    check_grouped(F.grouped_linear_fp8_blocks(x, sx, w, sw, i32(offsets), None, F32), x, sx, w, sw, offsets)


def test_a_groups_rows_do_not_depend_on_other_rows():
    """The same group with the same rows gives the same bits in another place among other groups."""
    w, sw = matrix(300, 1408, 1, 128, 3)
    x, sx = matrix(200, 1408, 2, 1)
    a = F.grouped_linear_fp8_blocks(x, sx, w, sw, i32([0, 40, 150, 200]))
    b = F.grouped_linear_fp8_blocks(x, sx, w, sw, i32([0, 40, 40, 200]), torch.arange(200, device=DEV).int())
    assert torch.equal(a[:40], b[:40]) and torch.equal(a[150:], b[150:])
    c = F.grouped_linear_fp8_blocks(x, sx, w, sw, i32([0, 40, 150, 200]))
    assert torch.equal(a, c)


def test_offsets_past_32_bits():
    """Rows of x, w and y whose byte offsets pass 2^31 and 2^32; few of each are looked at."""
    m, n, k = 70001, 33000, 160
    x, sx = matrix(m, k, 1, 1)
    w, sw = matrix(n, k, 2, 128)
    y = F.linear_fp8_blocks(x, sx, w, sw, BF)  # 4.6 GB
    at = torch.tensor([0, 1, 35000, 65077, 65078, m - 1], device=DEV)
    R.check_product(y[at], x.view(torch.uint8)[at].view(E4), sx[at], w, sw)
    del y
    far = 2 ** 27 + 16
    buf = torch.zeros(40 * far, dtype=torch.uint8, device=DEV)  # 5.4 GB
    wide = buf.view(40, far)[:, :k].view(E4)
    wide.view(torch.uint8).copy_(x[:40].view(torch.uint8))
    R.check_product(F.linear_fp8_blocks(wide, sx[:40], w[:300], sw[:3], F32), x[:40], sx[:40], w[:300], sw[:3])
    wide.view(torch.uint8).copy_(w[:40].view(torch.uint8))
    R.check_product(F.linear_fp8_blocks(x[:50], sx[:50], wide, sw[:1], F32), x[:50], sx[:50], w[:40], sw[:1])
    rows = torch.tensor([39, 0, 17, 38], device=DEV).int()
    wide.view(torch.uint8).copy_(x[:40].view(torch.uint8))
    got = F.grouped_linear_fp8_blocks(wide, sx[:40], w[:256].view(2, 128, k), sw[:2].view(2, 1, -1), i32([0, 2, 4]), rows, F32)
    check_grouped(got, x[:40], sx[:40], w[:256].view(2, 128, k), sw[:2].view(2, 1, -1), [0, 2, 4], rows)
    big = buf[:5 * 2 ** 30].view(BF).view(-1, 2560)  # 2^31 values and more
    big[-1] = rnd(2560, seed=4)
    codes, scales = F.quantize_fp8_blocks(big)
    q, s = R.rounded(big[-2:].double(), 1)
    R.check_codes(codes[-2:], q)
    R.check_scales(scales[-2:], s, U24)


# ---------------------------------------------------------------- as they are used
def layer(h, r, p, ids, offsets, rows):
    """An attention input and a routed MLP: what a layer with 8-bit weights calls."""
    c, s, h = F.rmsnorm_fp8_blocks(h, p["norm"], 1e-6, r)
    qkv = F.linear_fp8_blocks(c, s, p["w"], p["sw"])
    gu = F.grouped_linear_fp8_blocks(c, s, p["gu"], p["sgu"], offsets, rows)
    gate, up = gu.chunk(2, 1)
    a, sa = F.silu_mul_fp8_blocks(gate, up)
    y = F.grouped_linear_fp8_blocks(a, sa, p["down"], p["sdown"], offsets)
    return {"c": c, "s": s, "h": h, "qkv": qkv, "gu": gu, "a": a, "sa": sa, "y": y}


def layer_inputs(tokens, seed, hidden=512, inter=352, experts=8, top=3):
    p = {"norm": (1 + 0.2 * rnd(hidden, seed=9, dtype=F32)).to(BF)}
    p["w"], p["sw"] = matrix(700, hidden, 10, 128)
    p["gu"], p["sgu"] = matrix(2 * inter, hidden, 11, 128, experts)
    p["down"], p["sdown"] = matrix(hidden, inter, 12, 128, experts)
    h, r = rnd(tokens, hidden, seed=seed), rnd(tokens, hidden, seed=seed + 1)
    ids = torch.rand(tokens, experts, generator=gen(seed), device=DEV).topk(top, 1).indices.reshape(-1)
    order = torch.sort(ids, stable=True).indices
    counts = torch.bincount(ids, minlength=experts)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).int()
    return h, r, p, ids, offsets, (order // top).int()


def check_layer(o, h, r, p, ids, offsets, rows):
    """Each function's result against 64 bits from what it was given."""
    assert torch.equal(o["h"], (h.float() + r.float()).to(BF))
    hd = o["h"].double()
    q, s = R.rounded(hd * p["norm"].double(), 1)
    R.check_codes(o["c"], q)
    R.check_scales(o["s"], s / torch.sqrt((hd * hd).mean(1, keepdim=True) + 1e-6), 24 * U24)
    R.check_product(o["qkv"], o["c"], o["s"], p["w"], p["sw"])
    at = offsets.tolist()
    check_grouped(o["gu"], o["c"], o["s"], p["gu"], p["sgu"], at, rows)
    gate, up = o["gu"].double().chunk(2, 1)
    q, s = R.rounded(gate * torch.sigmoid(gate) * up, 1)
    R.check_codes(o["a"], q, 19 * U24)
    R.check_scales(o["sa"], s, 9 * U24)
    check_grouped(o["y"], o["a"], o["sa"], p["down"], p["sdown"], at)


@pytest.mark.parametrize("tokens", [1, 7, 64, 500])
def test_a_layer(tokens):
    args = layer_inputs(tokens, tokens)
    check_layer(layer(*args), *args)


def test_a_layer_captured_and_replayed_with_other_inputs():
    args = list(layer_inputs(24, 5))
    h, r, p, ids, offsets, rows = args
    layer(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(*args)
    for seed in (30, 31, 32):
        new = layer_inputs(24, seed)
        for a, b in zip((h, r, offsets, rows), (new[0], new[1], new[4], new[5])):
            a.copy_(b)
        graph.replay()
        eager = layer(h, r, p, new[3], offsets, rows)
        torch.cuda.synchronize()
        for name in out:
            assert torch.equal(out[name].view(torch.uint8), eager[name].view(torch.uint8)), name
        check_layer(out, h, r, p, new[3], offsets, rows)


def test_two_streams_at_once():
    a, b = layer_inputs(100, 1), layer_inputs(300, 2)
    want = [layer(*a), layer(*b)]
    torch.cuda.synchronize()
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for i, args in enumerate((a, b)):
            with torch.cuda.stream(s[i]):
                got[i].append(layer(*args))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            for name in o:
                assert torch.equal(o[name].view(torch.uint8), want[i][name].view(torch.uint8)), name


def test_more_leading_dimensions_and_single_rows():
    x = rnd(2, 3, 300, seed=1)
    w, sw = matrix(140, 300, 2, 128)
    norm = torch.ones(300, device=DEV, dtype=BF)
    for v in (x, x[0, 0], x[:, 1], x.transpose(0, 1)):
        flat = v.reshape(-1, 300)
        for got, want in ((F.quantize_fp8_blocks(v), F.quantize_fp8_blocks(flat)),
                          (F.silu_mul_fp8_blocks(v, v), F.silu_mul_fp8_blocks(flat, flat)),
                          (F.rmsnorm_fp8_blocks(v, norm, 1e-6, v), F.rmsnorm_fp8_blocks(flat, norm, 1e-6, flat))):
            for a, b in zip(got, want):
                assert a.shape[:-1] == v.shape[:-1]
                assert torch.equal(a.contiguous().view(torch.uint8).reshape(-1), b.view(torch.uint8).reshape(-1))
        c, s = F.quantize_fp8_blocks(v)
        y = F.linear_fp8_blocks(c, s, w, sw)
        assert y.shape == (*v.shape[:-1], 140)
        assert torch.equal(y.reshape(-1, 140), F.linear_fp8_blocks(*F.quantize_fp8_blocks(flat), w, sw))


def on_gpu(args):
    """Arguments of the refusal tests on the GPU, with their strides."""
    def there(a):
        if not isinstance(a, torch.Tensor):
            return a
        u = a.view(torch.uint8) if a.dtype.itemsize == 1 else a
        moved = torch.empty_strided(u.shape, u.stride(), dtype=u.dtype, device=DEV).zero_()
        return moved.view(a.dtype)
    return [there(a) for a in args]


@pytest.mark.parametrize("name,at,value,error,text", C.REFUSED)
def test_bad_arguments_are_refused_on_the_gpu_too(name, at, value, error, text):
    args = on_gpu(C.good()[name])
    getattr(F, name)(*args)
    args[at] = on_gpu([value])[0]
    with pytest.raises(error, match=text):
        getattr(F, name)(*args)


@pytest.mark.parametrize("name", sorted(C.good()))
def test_tensors_of_two_devices_are_refused(name):
    args = on_gpu(C.good()[name])
    for i, a in enumerate(args):
        if isinstance(a, torch.Tensor) and not (name == "quantize_fp8_blocks"):
            with pytest.raises((NotImplementedError, ValueError), match="requires CUDA|tensors on"):
                getattr(F, name)(*args[:i], a.cpu(), *args[i + 1:])


def test_the_plain_case_and_the_checks_one_by_one_agree(monkeypatch):
    """The head of each function and what follows it give the same."""
    args = layer_inputs(24, 5)
    want = layer(*args)
    monkeypatch.setattr(F, "_plain", lambda index: False)
    got = layer(*args)
    for name in want:
        assert torch.equal(got[name].view(torch.uint8), want[name].view(torch.uint8)), name


def test_weights_by_the_plain_case_and_by_the_checks_one_by_one(monkeypatch):
    x = torch.randn(300, 200, device=DEV, generator=gen(3))
    inputs = [x, x.to(BF), x[:, 3:], x[::2], x[:, :1], x.expand(1, 300, 200)[0]]
    w, sw = matrix(140, 300, 2, 128, 3)
    c, s = matrix(20, 300, 1, 1)
    rows = torch.tensor([3, 3, 19, 0, -1, 7, 20, 5, 5], device=DEV).int()

    def results():
        for v in inputs:
            yield from F.quantize_fp8_blocks(v, 128)
        for dtype in (None, BF, F32):
            yield F.grouped_linear_fp8_blocks(c, s, w, sw, i32([0, 4, 4, 20]), None, dtype)
            yield F.grouped_linear_fp8_blocks(c, s, w, sw, i32([0, 2, 9, 9]), rows, dtype)

    want = list(results())
    monkeypatch.setattr(F, "_plain", lambda index: False)
    for a, b in zip(results(), want):
        assert a.shape == b.shape and a.dtype == b.dtype and a.is_contiguous() and b.is_contiguous()
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_no_rows():
    w, sw = matrix(140, 300, 2, 128)
    x = torch.zeros(0, 300, device=DEV, dtype=BF)
    c, s = F.quantize_fp8_blocks(x)
    assert F.linear_fp8_blocks(c, s, w, sw).shape == (0, 140)
    assert F.rmsnorm_fp8_blocks(x, x.new_ones(300), 1e-6)[1].shape == (0, 3)
    assert F.silu_mul_fp8_blocks(x, x)[0].shape == (0, 300)
    assert F.grouped_linear_fp8_blocks(c, s, w[None], sw[None], i32([0, 0])).shape == (0, 140)
