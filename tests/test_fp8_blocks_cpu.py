"""The 8-bit functions with block scales without a GPU: what they and their entry points refuse, before any launch, and
the definition that the GPU tests hold them to."""

from __future__ import annotations

import math

import pytest
import torch

import fp8_blocks_ref as R
from triton_kernels import _hip
from triton_kernels import fp8_blocks as F

BF, E4 = torch.bfloat16, torch.float8_e4m3fn


def z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def codes(*shape):
    return torch.zeros(*shape, dtype=torch.uint8).view(E4)


def good():
    """Arguments that each function takes, by function."""
    return {
        "quantize_fp8_blocks": [z(5, 200, dtype=BF), 1],
        "rmsnorm_fp8_blocks": [z(5, 200, dtype=BF), z(200, dtype=BF), 1e-6, z(5, 200, dtype=BF)],
        "silu_mul_fp8_blocks": [z(5, 200, dtype=BF), z(5, 200, dtype=BF)],
        "linear_fp8_blocks": [codes(5, 200), z(5, 2), codes(300, 200), z(3, 2), BF],
        "grouped_linear_fp8_blocks": [codes(5, 200), z(5, 2), codes(4, 300, 200), z(4, 3, 2),
                                      z(5, dtype=torch.int32), z(7, dtype=torch.int32), BF],
    }


@pytest.mark.parametrize("name", sorted(good()))
def test_functions_refuse_cpu_tensors(name):
    with pytest.raises(NotImplementedError, match="requires CUDA"):
        getattr(F, name)(*good()[name])


REFUSED = [
    ("quantize_fp8_blocks", 0, z(5, 200, dtype=torch.float16), NotImplementedError, "bf16 or fp32"),
    ("quantize_fp8_blocks", 0, z(5, 0, dtype=BF), ValueError, r"x is \[5, 0\]"),
    ("quantize_fp8_blocks", 0, z(200, 5, dtype=BF).T, NotImplementedError, "contiguous last"),
    ("quantize_fp8_blocks", 0, z(()), ValueError, "must have rows"),
    ("quantize_fp8_blocks", 1, 64, ValueError, "block_rows must be 1 or 128"),
    ("rmsnorm_fp8_blocks", 0, z(5, 200, dtype=torch.float64), NotImplementedError, "bf16 or fp32"),
    ("rmsnorm_fp8_blocks", 1, z(200), NotImplementedError, "weight is"),
    ("rmsnorm_fp8_blocks", 1, z(199, dtype=BF), ValueError, "weight shape"),
    ("rmsnorm_fp8_blocks", 1, z(400, dtype=BF)[::2], NotImplementedError, "weight must be contiguous"),
    ("rmsnorm_fp8_blocks", 2, -1e-6, ValueError, "eps"),
    ("rmsnorm_fp8_blocks", 2, math.nan, ValueError, "eps"),
    ("rmsnorm_fp8_blocks", 2, math.inf, ValueError, "eps"),
    ("rmsnorm_fp8_blocks", 3, z(5, 200), NotImplementedError, "residual is"),
    ("rmsnorm_fp8_blocks", 3, z(200, dtype=BF), ValueError, "residual is"),
    ("silu_mul_fp8_blocks", 1, z(5, 201, dtype=BF), ValueError, "same shape"),
    ("silu_mul_fp8_blocks", 1, z(5, 200), NotImplementedError, "up torch.float32"),
    ("silu_mul_fp8_blocks", 1, z(200, 5, dtype=BF).T, NotImplementedError, "contiguous last"),
    ("linear_fp8_blocks", 0, z(5, 200, dtype=torch.uint8), NotImplementedError, "float8_e4m3fn"),
    ("linear_fp8_blocks", 0, z(5, 200).to(torch.float8_e5m2), NotImplementedError, "float8_e4m3fn"),
    ("linear_fp8_blocks", 1, z(5, 1), ValueError, "x_scales must be"),
    ("linear_fp8_blocks", 1, z(4, 2), ValueError, "x_scales must be"),
    ("linear_fp8_blocks", 1, z(2, 5).T, NotImplementedError, "contiguous last"),
    ("linear_fp8_blocks", 1, z(5, 2, dtype=BF), NotImplementedError, "x_scales must be fp32"),
    ("linear_fp8_blocks", 2, codes(300, 199), ValueError, "weights must be"),
    ("linear_fp8_blocks", 2, codes(0, 200), ValueError, "weights must be"),
    ("linear_fp8_blocks", 2, codes(4, 300, 200), ValueError, "weights must be"),
    ("linear_fp8_blocks", 2, codes(200, 300).T, NotImplementedError, "contiguous last"),
    ("linear_fp8_blocks", 2, z(300, 200, dtype=BF), NotImplementedError, "float8_e4m3fn"),
    ("linear_fp8_blocks", 3, z(2, 2), ValueError, "weight scales must be"),
    ("linear_fp8_blocks", 3, z(3, 2).double(), NotImplementedError, "weight scales must be fp32"),
    ("linear_fp8_blocks", 4, torch.float16, NotImplementedError, "output_dtype"),
    ("grouped_linear_fp8_blocks", 0, codes(5, 1, 200), ValueError, "x must be"),
    ("grouped_linear_fp8_blocks", 2, codes(300, 200), ValueError, "weights must be"),
    ("grouped_linear_fp8_blocks", 3, z(4, 2, 3), ValueError, "weight scales must be"),
    ("grouped_linear_fp8_blocks", 4, z(4, dtype=torch.int32), ValueError, "offsets must be"),
    ("grouped_linear_fp8_blocks", 4, z(5, dtype=torch.int64), NotImplementedError, "int32"),
    ("grouped_linear_fp8_blocks", 4, z(10, dtype=torch.int32)[::2], NotImplementedError, "contiguous"),
    ("grouped_linear_fp8_blocks", 5, z(7, dtype=torch.int64), NotImplementedError, "int32"),
    ("grouped_linear_fp8_blocks", 5, z(7, 1, dtype=torch.int32), ValueError, "rows"),
    ("grouped_linear_fp8_blocks", 5, z(14, dtype=torch.int32)[::2], NotImplementedError, "contiguous"),
]


@pytest.mark.parametrize("name,at,value,error,text", REFUSED)
def test_functions_refuse_bad_arguments_before_any_launch(monkeypatch, name, at, value, error, text):
    monkeypatch.setattr(F, "_device", lambda *a: 0)
    calls = []
    monkeypatch.setattr(F, "_call", lambda index, entry, *args: calls.append(entry))
    getattr(F, name)(*good()[name])
    assert len(calls) == 1
    args = good()[name]
    args[at] = value
    with pytest.raises(error, match=text):
        getattr(F, name)(*args)
    assert len(calls) == 1


def test_results_have_the_shapes_that_the_next_function_takes(monkeypatch):
    monkeypatch.setattr(F, "_device", lambda *a: 0)
    calls = []
    monkeypatch.setattr(F, "_call", lambda index, entry, *args: calls.append(entry))
    for lead in [(), (1,), (7,), (2, 3), (0,), (2, 0)]:
        x = z(*lead, 300, dtype=BF)
        for out in (F.quantize_fp8_blocks(x), F.silu_mul_fp8_blocks(x, x), F.rmsnorm_fp8_blocks(x, z(300, dtype=BF), 0.0)):
            assert out[0].shape == x.shape and out[0].dtype == E4
            assert out[1].shape == (*lead, 3) and out[1].dtype == torch.float32
            y = F.linear_fp8_blocks(*out, codes(40, 300), z(1, 3))
            assert y.shape == (*lead, 40) and y.dtype == BF
        c, s, h = F.rmsnorm_fp8_blocks(x, z(300, dtype=BF), 0.0, x)
        assert h.shape == x.shape and h.dtype == BF
    del calls[:]
    for shape, scales in [((130, 300), (2, 3)), ((4, 130, 300), (4, 2, 3)), ((1, 1), (1, 1)), ((0, 8), (0, 1)),
                          ((0, 8, 8), (0, 1, 1)), ((3, 0, 8), (3, 0, 1))]:
        c, s = F.quantize_fp8_blocks(z(*shape), 128)
        assert c.shape == shape and s.shape == scales
    assert len(calls) == 3  # nothing is launched for nothing
    y = F.grouped_linear_fp8_blocks(codes(5, 200), z(5, 2), codes(4, 300, 200), z(4, 3, 2), z(5, dtype=torch.int32))
    assert y.shape == (5, 300)
    y = F.grouped_linear_fp8_blocks(codes(0, 200), z(0, 2), codes(4, 300, 200), z(4, 3, 2), z(5, dtype=torch.int32),
                                    z(9, dtype=torch.int32), torch.float32)
    assert y.shape == (9, 300) and y.dtype == torch.float32


def test_entry_points_refuse_bad_arguments_without_launching():
    one = 1 << 20  # never read: every call below is refused on the host

    def refused(entry, args, *bad):
        for at, value, match in bad:
            with pytest.raises(_hip.HipKernelError, match=match):
                _hip.call(entry, *args[:at], value, *args[at + 1:], None)

    refused("dsv2_quantize_fp8_blocks", [one, 200, 0, 1, 5, 200, 0, 1, one, one],
            (0, None, "null"), (0, one + 1, "alignment"), (1, -8, "alignment"), (3, 2, "groups"), (4, -1, "rows"),
            (5, 0, "rows"), (5, 2 ** 31 - 1, "rows"), (6, 2, "dtype"), (7, 64, "blocks of 64"), (8, None, "null"),
            (9, one + 2, "alignment"), (4, 2 ** 40, "rows"), (5, 2 ** 30 + 1, "rows of"))
    refused("dsv2_quantize_fp8_blocks", [one, 200, 0, 1, 5, 200, 1, 128, one, one],
            (0, one + 2, "alignment"), (4, 2 ** 40, "matrices"), (3, 2 ** 31, "matrices"), (3, -1, "groups"))
    refused("dsv2_rmsnorm_fp8_blocks", [one, 200, one, 200, one, 1e-6, 5, 200, 0, one, one, one],
            (0, None, "null"), (4, None, "null"), (11, None, "null"), (9, None, "null"), (6, 2 ** 31, "rows"),
            (7, 0, "rows"), (7, 2 ** 30 + 1, "rows of"), (8, 3, "dtype"), (4, one + 1, "alignment"), (11, one + 1, "alignment"))
    refused("dsv2_silu_mul_fp8_blocks", [one, 200, one, 200, 5, 200, 0, one, one],
            (0, None, "null"), (2, None, "null"), (2, one + 1, "alignment"), (4, -1, "rows"), (4, 2 ** 40, "rows"),
            (5, 2 ** 30 + 1, "rows of"), (6, -1, "dtype"))
    product = [one, 200, one, 2, 5, 200, one, 200, one, 2, 300, one, 300, 0]
    refused("dsv2_linear_fp8_blocks", product,
            (0, None, "null"), (2, one + 2, "alignment"), (4, -1, "rows"), (4, 2 ** 31, "rows"), (5, 0, "K 0"), (5, 2 ** 30 + 1, "K"), (10, 2 ** 30 + 1, "N"),
            (8, None, "null"), (10, 0, "N 0"), (11, one + 1, "alignment"), (12, 299, "strides"), (7, -1, "strides"),
            (13, 2, "out_dtype"))
    with pytest.raises(_hip.HipKernelError, match="rows of"):  # more tiles than a launch has workgroups
        _hip.call("dsv2_linear_fp8_blocks", one, 200, one, 2, 2 ** 31 - 1, 200, one, 200, one, 2, 2 ** 30, one, 2 ** 30, 0,
                  None)
    grouped = [one, 200, one, 2, 5, one, 7, 200, one, 60000, 200, one, 6, 2, 300, 4, one, one, 300, 1]
    refused("dsv2_grouped_linear_fp8_blocks", grouped,
            (0, None, "null"), (4, -1, "rows of x"), (5, None, "rows of x"), (5, one + 2, "alignment"), (6, -1, "rows"),
            (9, -1, "strides"), (15, 0, "0 groups"), (15, 65537, "groups"), (16, None, "null"), (17, one + 2, "alignment"))


@pytest.mark.parametrize("rows,k,n,groups,f32", [(600_000_000, 16, 16, 0, 1), (1_000_000_000, 1, 3, 0, 0), (1, 16, 2 ** 30, 0, 0),
                                                 (1, 16, 2 ** 30, 1, 1), (65536, 16, 30_000, 65536, 0)])
def test_calls_of_very_many_tiles_take_tiles_that_a_launch_has_room_for(rows, k, n, groups, f32):
    shape = _hip.lib.dsv2_linear_fp8_blocks_tiles(rows, k, n, groups, f32)
    bm, bn, threads = {0: (16, 16, 512), 1: (32, 16, 512), 2: (32, 32, 256), 3: (32, 64, 128), 4: (64, 64, 512),
                       5: (128, 64, 512), 6: (128, 128, 512), 7: (128, 256, 512), 8: (256, 256, 512), 10: (16, 32, 64),
                       11: (16, 16, 512), 13: (32, 32, 256), 15: (64, 64, 512), 17: (128, 128, 512)}[shape]
    tiles = (rows + min(rows, groups) * (bm - 1)) // bm if groups else -(-rows // bm)
    assert tiles * -(-n // bn) * threads < 2 ** 32


# kernel: tokens and features of a tile, threads of a workgroup (kernel 7: with bf16 and with fp32 results)
TILES = {0: (16, 16, 512), 1: (32, 16, 512), 2: (32, 32, 256), 3: (32, 64, 128), 4: (64, 64, 512), 5: (128, 64, 512),
         6: (128, 128, 512), 7: (128, 256, (1024, 512)), 8: (256, 256, 512), 10: (16, 32, 64), 11: (16, 16, 512),
         13: (32, 32, 256), 15: (64, 64, 512), 17: (128, 128, 512)}


def room(shape, rows, n, groups, f32):
    """Workgroups that the kernel has, and that a launch of its workgroups has room for (beyond 2^32 threads there are none;
    a launch is rounded up to eights)."""
    bm, bn, threads = TILES[shape]
    threads = threads if isinstance(threads, int) else threads[f32]
    tiles = (rows + min(rows, groups) * (bm - 1)) // bm if groups else -(-rows // bm)
    return tiles * -(-n // bn), 2 ** 32 // threads - 8


@pytest.mark.parametrize("rows,k,n,groups,f32", [(1114112, 512, 14400, 65536, 0), (2 ** 21, 16, 13312, 65536, 0),
                                                 (2 ** 20, 16, 20000, 65536, 0), (2 ** 20, 16, 20000, 65536, 1),
                                                 (2 ** 20, 16, 16000, 65536, 1), (1114112, 512, 14400, 65536, 1)])
def test_the_kernel_of_a_huge_grouped_call_is_one_that_a_launch_has_room_for(rows, k, n, groups, f32):
    """Where some kernel has room, the one that is taken has it."""
    shape = _hip.lib.dsv2_linear_fp8_blocks_tiles(rows, k, n, groups, f32)
    able = []
    for s in TILES:
        needed, most = room(s, rows, n, groups, f32)
        if s < 11 and not (s == 8 and (f32 or k <= 128)) and needed <= most:
            able.append(s)
    assert able and shape in able


@pytest.mark.parametrize("args", [(0, 128, 128, 0, 0), (-1, 128, 128, 0, 0), (2 ** 31, 128, 128, 0, 0), (5, 0, 128, 0, 0),
                                  (5, -16, 128, 2, 0), (5, 128, 0, 0, 1), (5, 2 ** 30 + 1, 128, 0, 0), (5, 128, 128, -1, 0),
                                  (5, 128, 128, 65537, 0)])
def test_the_tiles_of_sizes_that_no_product_has_are_an_error(args):
    assert _hip.lib.dsv2_linear_fp8_blocks_tiles(*args) == -2


def test_definition_of_the_rounding():
    """The 64-bit form against torch's conversion, and against every code and every tie."""
    q = torch.arange(256, dtype=torch.uint8).view(E4).float()
    q = q[q.isfinite()].double().sort().values.unique()
    assert torch.equal(R.nearest(q)[0], q) and q.max() == 448
    mid = (q[1:] + q[:-1]) / 2
    for v in (q, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20)):
        assert torch.equal(R.nearest(v)[0], v.float().to(E4).double())
    quotients, scales = R.rounded(torch.tensor([[448.0, -3.0, 0.0], [0.0, 0.0, 0.0], [1.0, math.nan, 2.0]]).double(), 1)
    assert torch.equal(quotients[0], torch.tensor([448.0, -3.0, 0.0]).double()) and scales[0] == 1
    assert not quotients[1].any() and scales[1] == 2.0 ** -100 / 448
    assert quotients[2].isnan().all() and scales[2].isnan()
