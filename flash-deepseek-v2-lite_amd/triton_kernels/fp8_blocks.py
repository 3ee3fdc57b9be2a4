"""8-bit floating point with a scale for each block of 128: rounding of activations and weights, RMSNorm and
SwiGLU that end in it, and the matrix products of what comes out, dense and grouped by experts.

No counterpart in the reference (bf16 throughout); these stand beside ``rmsnorm``, ``mlp_elementwise`` and
``moe_batch`` for models whose weights come as e4m3 codes with a fp32 scale for each 128 x 128 block.

Codes are OCP e4m3 (``torch.float8_e4m3fn``).  A block is 128 columns (the last one of a row may be shorter) of one
row of activations or of 128 rows of weights.  With a its largest |v|, at least 2^-100, its scale is a / 448 and
its codes are the e4m3 values nearest to 448 v / a, ties to even; a block with an infinity or a NaN stands for NaN
throughout.  Activations [..., K] come with scales [..., ceil(K / 128)], weights [(E,) N, K] with scales
[(E,) ceil(N / 128), ceil(K / 128)].

Every function runs on its tensors' device and that device's current stream, takes no workspace and reads
nothing back to the host: all may be captured into a graph.  Last dimensions have to be contiguous, rows may be any
stride apart; whole 16-byte rows are read faster.

Products with fp32 results are sums in fp32.  bf16 results (the default) take the 8-bit matrix instruction for the sum
within a block: it aligns the products of 8 neighbouring columns to the largest of them and drops what lies 2^-13 below
it, 1.3e-5 of the sum for normal values.  Where large terms cancel that can be more than bf16's rounding of what is left:
ask for fp32 results there.  Blocks are added up in fp32 either way.
"""

from __future__ import annotations

import math

import torch

from . import _hip

BLOCK = 128
MAX_ROWS = 2 ** 31 - 1
MAX_COLS = 2 ** 30  # and features of a product
MAX_GROUPS = 65536

# These calls launch kernels of 2 to 10 us for few rows, so their own host time is looked at: a launch takes 3 us of it,
# an attribute of a tensor 0.05 to 0.1, new_empty 1.5, torch's allocation by shape, strides and type alone 0.7.  The
# plain case (matrices, as they should be, on the current device) is therefore found by one condition at the head of a
# function; whatever does not meet it goes through the checks one by one.
_E4M3, _BF16, _F32, _I32 = torch.float8_e4m3fn, torch.bfloat16, torch.float32, torch.int32
_TYPES = {_BF16: 0, _F32: 1}  # DSV2_DTYPE_*
_ENTRY = {n: getattr(_hip.lib, n) for n in ("dsv2_quantize_fp8_blocks", "dsv2_rmsnorm_fp8_blocks",
                                            "dsv2_silu_mul_fp8_blocks", "dsv2_linear_fp8_blocks",
                                            "dsv2_grouped_linear_fp8_blocks")}
_QUANTIZE, _RMSNORM, _SILU, _LINEAR, _GROUPED = _ENTRY.values()
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_empty_strided = getattr(getattr(getattr(torch._C, "_dynamo", None), "guards", None), "_empty_strided_cuda", None)


def _check(rc: int, entry: str) -> None:
    if rc:
        raise _hip.HipKernelError(f"{entry} failed (status {rc}): "
                                  f"{_hip.lib.dsv2_last_error_message().decode(errors='replace')}")


def _plain(index: int) -> bool:
    """Tensors of that device may be allocated and used without a change of the current one."""
    return index >= 0 and _empty_strided is not None and _current_device() == index


def _call(index: int, entry: str, *args) -> None:
    """The entry point on the device's current stream, with the device as the current one."""
    if _current_device() != index:
        with torch.cuda.device(index):
            return _call(index, entry, *args)
    _check(_ENTRY[entry](*args, _hip._raw_stream(index)), entry)


def _device(name: str, *ts: torch.Tensor) -> int:
    """The index of the one GPU that all tensors are on."""
    index = ts[0].get_device()
    for t in ts:
        if t.get_device() != index or index < 0:
            if not t.is_cuda:
                raise NotImplementedError(f"{name} requires CUDA (HIP) tensors")
            raise ValueError(f"{name}: tensors on {ts[0].device} and {t.device}")
    return index


def _matrix(like: torch.Tensor, n: int, k: int, dtype: torch.dtype) -> torch.Tensor:
    """An uninitialised [n, k] on the device of `like`."""
    return like.new_empty((n, k), dtype=dtype)


def _type(name: str, what: str, t: torch.Tensor) -> int:
    code = _TYPES.get(t.dtype)
    if code is None:
        raise NotImplementedError(f"{name}: {what} must be bf16 or fp32, not {t.dtype}")
    return code


def _rows(name: str, what: str, t: torch.Tensor) -> tuple[torch.Tensor, int, int, int]:
    """(t as a matrix, its rows, its columns, its row stride)."""
    shape = t.shape
    if len(shape) != 2:
        if not shape:
            raise ValueError(f"{name}: {what} must have rows, not be a number")
        t = t.reshape(math.prod(shape[:-1]), shape[-1])
        shape = t.shape
    n, k = shape
    rs, cs = t.stride()
    if k == 0 or n > MAX_ROWS or k > MAX_COLS:
        raise ValueError(f"{name}: {what} is {list(shape)}")
    if cs != 1 and k > 1:
        raise NotImplementedError(f"{name}: {what} must have a contiguous last dimension")
    return t, n, k, rs


def _shaped(like: torch.Tensor, *results: torch.Tensor) -> tuple[torch.Tensor, ...]:
    """Matrices with the leading dimensions of `like`."""
    lead = like.shape[:-1]
    return results if len(lead) == 1 else tuple(r.view(*lead, r.shape[1]) for r in results)


def quantize_fp8_blocks(x: torch.Tensor, block_rows: int = 1) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of bf16 or fp32 values: activations [..., K] in blocks of one row (``block_rows`` 1) or weights
    [N, K] or [E, N, K] in blocks of 128 rows (``block_rows`` 128; a matrix's last block may be shorter)."""
    name = "quantize_fp8_blocks"
    if x.dim() == 2 and (block_rows == 1 or block_rows == BLOCK):
        n, k = x.shape
        rs, cs = x.stride()
        dtype, index = _TYPES.get(x.dtype), x.get_device()
        if dtype is not None and cs == 1 and 0 < n <= MAX_ROWS and 0 < k <= MAX_COLS and _plain(index):
            kb, nb = (k + 127) // BLOCK, n if block_rows == 1 else (n + 127) // BLOCK
            codes, scales = _empty_strided((n, k), (k, 1), _E4M3), _empty_strided((nb, kb), (kb, 1), _F32)
            _check(_QUANTIZE(x.data_ptr(), rs, 0, 1, n, k, dtype, block_rows, codes.data_ptr(), scales.data_ptr(),
                             _hip._raw_stream(index)), name)
            return codes, scales
    index = _device(name, x)
    dtype = _type(name, "x", x)
    if block_rows == 1:
        m, n, k, rs = _rows(name, "x", x)
        codes, scales = _matrix(m, n, k, _E4M3), _matrix(m, n, (k + 127) // BLOCK, _F32)
        if n:
            _call(index, "dsv2_quantize_fp8_blocks", m.data_ptr(), rs, 0, 1, n, k, dtype, 1, codes.data_ptr(),
                  scales.data_ptr())
        return _shaped(x, codes, scales)
    if block_rows == BLOCK:
        if x.dim() not in (2, 3):
            raise ValueError(f"{name}: weights must be [N, K] or [E, N, K], not {list(x.shape)}")
        groups, gs = (1, 0) if x.dim() == 2 else (x.shape[0], x.stride(0))
        n, k = x.shape[-2:]
        rs, cs = x.stride()[-2:]
        if k == 0 or max(n, groups) > MAX_ROWS or k > MAX_COLS:
            raise ValueError(f"{name}: x is {list(x.shape)}")
        if cs != 1 and k > 1:
            raise NotImplementedError(f"{name}: x must have a contiguous last dimension")
        codes = x.new_empty(x.shape, dtype=_E4M3)
        scales = x.new_empty((*x.shape[:-2], -(-n // BLOCK), -(-k // BLOCK)), dtype=_F32)
    else:
        raise ValueError(f"{name}: block_rows must be 1 or {BLOCK}, not {block_rows}")
    if n and groups:
        _call(index, "dsv2_quantize_fp8_blocks", x.data_ptr(), rs, gs, groups, n, k, dtype, BLOCK, codes.data_ptr(),
              scales.data_ptr())
    return codes, scales


def rmsnorm_fp8_blocks(hidden_states: torch.Tensor, weight: torch.Tensor, eps: float,
                       residual: torch.Tensor | None = None) -> tuple[torch.Tensor, ...]:
    """(codes, scales) of h * weight / sqrt(mean(h^2) + eps) over the last dimension, h = ``hidden_states``; with a
    ``residual`` of the same shape h is their sum, rounded to the inputs' type, and the third result.

    bf16 or fp32, all of one type; fp32 inside, and nothing is rounded between the norm and the codes (``rmsnorm_triton``
    rounds twice there).  The least block, 2^-100, is one of h * weight here."""
    name = "rmsnorm_fp8_blocks"
    x, index = hidden_states, hidden_states.get_device()
    if x.dim() == 2 and _plain(index) and weight.get_device() == index:
        n, k = x.shape
        rs, cs = x.stride()
        dtype, t = x.dtype, _TYPES.get(x.dtype)
        if (t is not None and cs == 1 and 0 < n <= MAX_ROWS and 0 < k <= MAX_COLS and 0.0 <= eps < math.inf and
                weight.dtype is dtype and weight.shape == (k,) and weight.is_contiguous()):
            kb = (k + 127) // BLOCK
            if residual is None:
                codes, scales = _empty_strided((n, k), (k, 1), _E4M3), _empty_strided((n, kb), (kb, 1), _F32)
                _check(_RMSNORM(x.data_ptr(), rs, None, 0, weight.data_ptr(), eps, n, k, t, codes.data_ptr(),
                                scales.data_ptr(), None, _hip._raw_stream(index)), name)
                return codes, scales
            if (residual.dtype is dtype and residual.get_device() == index and residual.shape == (n, k) and
                    residual.stride(1) == 1):
                codes, scales = _empty_strided((n, k), (k, 1), _E4M3), _empty_strided((n, kb), (kb, 1), _F32)
                total = _empty_strided((n, k), (k, 1), dtype)
                _check(_RMSNORM(x.data_ptr(), rs, residual.data_ptr(), residual.stride(0), weight.data_ptr(), eps, n, k, t,
                                codes.data_ptr(), scales.data_ptr(), total.data_ptr(), _hip._raw_stream(index)), name)
                return codes, scales, total
    index = _device(name, hidden_states, weight) if residual is None else _device(name, hidden_states, weight, residual)
    dtype = _type(name, "hidden_states", hidden_states)
    x, n, k, rs = _rows(name, "hidden_states", hidden_states)
    if weight.dtype is not hidden_states.dtype:
        raise NotImplementedError(f"{name}: weight is {weight.dtype}, hidden_states {hidden_states.dtype}")
    if weight.shape != (k,):
        raise ValueError(f"weight shape {tuple(weight.shape)} != ({k},)")
    if not weight.is_contiguous():
        raise NotImplementedError(f"{name}: weight must be contiguous")
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"{name}: eps must be at least 0 and finite, not {eps}")
    codes, scales = _matrix(x, n, k, _E4M3), _matrix(x, n, (k + 127) // BLOCK, _F32)
    if residual is None:
        if n:
            _call(index, "dsv2_rmsnorm_fp8_blocks", x.data_ptr(), rs, None, 0, weight.data_ptr(), eps, n, k, dtype,
                  codes.data_ptr(), scales.data_ptr(), None)
        return _shaped(hidden_states, codes, scales)
    if residual.dtype is not hidden_states.dtype:
        raise NotImplementedError(f"{name}: residual is {residual.dtype}, hidden_states {hidden_states.dtype}")
    if residual.shape != hidden_states.shape:
        raise ValueError(f"{name}: residual is {list(residual.shape)}, hidden_states {list(hidden_states.shape)}")
    res, _, _, res_stride = _rows(name, "residual", residual)
    total = _matrix(x, n, k, x.dtype)
    if n:
        _call(index, "dsv2_rmsnorm_fp8_blocks", x.data_ptr(), rs, res.data_ptr(), res_stride, weight.data_ptr(), eps, n, k,
              dtype, codes.data_ptr(), scales.data_ptr(), total.data_ptr())
    return _shaped(hidden_states, codes, scales, total)


def silu_mul_fp8_blocks(gate: torch.Tensor, up: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of silu(gate) * up, bf16 or fp32 [..., K] each (the halves of one gate_up result, as views);
    fp32 inside, nothing is rounded before the codes."""
    name = "silu_mul_fp8_blocks"
    index = gate.get_device()
    if gate.dim() == 2 and up.dim() == 2 and _plain(index) and up.get_device() == index:
        n, k = shape = gate.shape
        (gs, gc), (us, uc), t = gate.stride(), up.stride(), _TYPES.get(gate.dtype)
        if (t is not None and up.dtype is gate.dtype and up.shape == shape and gc == uc == 1 and 0 < n <= MAX_ROWS and
                0 < k <= MAX_COLS):
            kb = (k + 127) // BLOCK
            codes, scales = _empty_strided((n, k), (k, 1), _E4M3), _empty_strided((n, kb), (kb, 1), _F32)
            _check(_SILU(gate.data_ptr(), gs, up.data_ptr(), us, n, k, t, codes.data_ptr(), scales.data_ptr(),
                         _hip._raw_stream(index)), name)
            return codes, scales
    index = _device(name, gate, up)
    if gate.shape != up.shape:
        raise ValueError("gate and up must have the same shape")
    dtype = _type(name, "gate", gate)
    if up.dtype != gate.dtype:
        raise NotImplementedError(f"{name}: gate is {gate.dtype}, up {up.dtype}")
    g, n, k, gs = _rows(name, "gate", gate)
    u, _, _, us = _rows(name, "up", up)
    codes, scales = _matrix(g, n, k, _E4M3), _matrix(g, n, (k + 127) // BLOCK, _F32)
    if n:
        _call(index, "dsv2_silu_mul_fp8_blocks", g.data_ptr(), gs, u.data_ptr(), us, n, k, dtype, codes.data_ptr(),
              scales.data_ptr())
    return _shaped(gate, codes, scales)


def _activations(name: str, x: torch.Tensor, scales: torch.Tensor) -> tuple[torch.Tensor, int, int, int, torch.Tensor, int]:
    """(x as a matrix, rows, K, row stride, the scales as a matrix, their row stride)."""
    if x.dtype is not _E4M3:
        raise NotImplementedError(f"{name}: x must be float8_e4m3fn codes, not {x.dtype}")
    if scales.dtype is not _F32:
        raise NotImplementedError(f"{name}: x_scales must be fp32")
    codes, n, k, rs = _rows(name, "x", x)
    want = (*x.shape[:-1], (k + 127) // BLOCK)
    if scales.shape != want:
        raise ValueError(f"{name}: x_scales must be {list(want)}, not {list(scales.shape)}")
    scales, _, _, ss = _rows(name, "x_scales", scales)
    return codes, n, k, rs, scales, ss


def _weights(name: str, w: torch.Tensor, scales: torch.Tensor, k: int, dims: int) -> tuple[tuple[int, ...], ...]:
    """(shape, strides, the scales' strides)."""
    if w.dtype is not _E4M3:
        raise NotImplementedError(f"{name}: weights must be float8_e4m3fn codes, not {w.dtype}")
    if scales.dtype is not _F32:
        raise NotImplementedError(f"{name}: weight scales must be fp32")
    shape = w.shape
    if len(shape) != dims or shape[-1] != k or 0 in shape or shape[-2] > MAX_COLS:
        raise ValueError(f"{name}: weights must be {'[E, ' if dims == 3 else '['}N, {k}], not {list(shape)}")
    want = (*shape[:-2], (shape[-2] + 127) // BLOCK, (k + 127) // BLOCK)
    if scales.shape != want:
        raise ValueError(f"{name}: weight scales must be {list(want)}, not {list(scales.shape)}")
    strides, scale_strides = w.stride(), scales.stride()
    if strides[-1] != 1 and k > 1 or scale_strides[-1] != 1 and want[-1] > 1:
        raise NotImplementedError(f"{name}: weights and their scales must have a contiguous last dimension")
    return shape, strides, scale_strides


def _out_type(name: str, dtype: torch.dtype | None) -> tuple[torch.dtype, int]:
    if dtype is None:
        return _BF16, 0
    if dtype not in _TYPES:
        raise NotImplementedError(f"{name}: output_dtype must be bf16 or fp32")
    return dtype, _TYPES[dtype]


def linear_fp8_blocks(x: torch.Tensor, x_scales: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor,
                      output_dtype: torch.dtype | None = None) -> torch.Tensor:
    """The product [..., N] of activations [..., K] (codes, scales) and weights [N, K] (codes, scales), rounded once to
    ``output_dtype`` (bf16, the default, or fp32).  Sums are in fp32, for bf16 results with a narrower adder inside a block
    (above): large terms that cancel need fp32 results.  A block's two scales are multiplied first, in fp32: their product
    has to be in its range."""
    name = "linear_fp8_blocks"
    index = x.get_device()
    if (x.dim() == 2 and x_scales.dim() == 2 and weight.dim() == 2 and weight_scales.dim() == 2 and _plain(index) and
            x_scales.get_device() == index and weight.get_device() == index and weight_scales.get_device() == index):
        n, k = x.shape
        out, wk = weight.shape
        kb, t = (k + 127) // BLOCK, 0 if output_dtype is None else _TYPES.get(output_dtype)
        (xs, xc), (xss, xsc), (ws, wc), (wss, wsc) = x.stride(), x_scales.stride(), weight.stride(), weight_scales.stride()
        if (x.dtype is _E4M3 and weight.dtype is _E4M3 and x_scales.dtype is _F32 and weight_scales.dtype is _F32 and
                t is not None and wk == k and xc == wc == xsc == wsc == 1 and 0 < n <= MAX_ROWS and 0 < k <= MAX_COLS and
                0 < out <= MAX_COLS and x_scales.shape == (n, kb) and weight_scales.shape == ((out + 127) // BLOCK, kb)):
            y = _empty_strided((n, out), (out, 1), output_dtype or _BF16)
            _check(_LINEAR(x.data_ptr(), xs, x_scales.data_ptr(), xss, n, k, weight.data_ptr(), ws, weight_scales.data_ptr(),
                           wss, out, y.data_ptr(), out, t, _hip._raw_stream(index)), name)
            return y
    index = _device(name, x, x_scales, weight, weight_scales)
    codes, n, k, xs, x_scales, xss = _activations(name, x, x_scales)
    (out, _), (ws, _), (wss, _) = _weights(name, weight, weight_scales, k, 2)
    dtype, code = _out_type(name, output_dtype)
    y = _matrix(codes, n, out, dtype)
    if n:
        _call(index, "dsv2_linear_fp8_blocks", codes.data_ptr(), xs, x_scales.data_ptr(), xss, n, k, weight.data_ptr(), ws,
              weight_scales.data_ptr(), wss, out, y.data_ptr(), out, code)
    return _shaped(x, y)[0]


def grouped_linear_fp8_blocks(x: torch.Tensor, x_scales: torch.Tensor, weights: torch.Tensor, weight_scales: torch.Tensor,
                              offsets: torch.Tensor, rows: torch.Tensor | None = None,
                              output_dtype: torch.dtype | None = None) -> torch.Tensor:
    """The products [R, N] of rows sorted by group (expert): rows offsets[e] .. offsets[e + 1] are multiplied by
    ``weights[e]`` of [E, N, K].  Row r is row r of ``x`` [R, K], or row ``rows[r]`` of ``x`` [T, K] (int32 [R]; a
    row number outside x stands for zeros).  Sums are those of ``linear_fp8_blocks``.

    ``offsets`` int32 [E + 1] is read on the device only.  Rows of no group are not written (here: undefined); an
    offset below the largest one before it, or outside [0, R], counts as the nearest that is not."""
    name = "grouped_linear_fp8_blocks"
    index = x.get_device()
    if (x.dim() == 2 and x_scales.dim() == 2 and weights.dim() == 3 and weight_scales.dim() == 3 and offsets.dim() == 1 and
            _plain(index) and x_scales.get_device() == index and weights.get_device() == index and
            weight_scales.get_device() == index and offsets.get_device() == index and
            (rows is None or rows.get_device() == index and rows.dim() == 1)):
        (r, k), (groups, out, wk) = x.shape, weights.shape
        n = r if rows is None else rows.shape[0]
        kb, t = (k + 127) // BLOCK, 0 if output_dtype is None else _TYPES.get(output_dtype)
        (xs, xc), (xss, xsc) = x.stride(), x_scales.stride()
        (wgs, ws, wc), (wsgs, wss, wsc) = weights.stride(), weight_scales.stride()
        if (x.dtype is _E4M3 and weights.dtype is _E4M3 and x_scales.dtype is _F32 and weight_scales.dtype is _F32 and
                offsets.dtype is _I32 and t is not None and wk == k and xc == wc == xsc == wsc == 1 and
                0 < n <= MAX_ROWS and 0 < r <= MAX_ROWS and 0 < k <= MAX_COLS and 0 < out <= MAX_COLS and
                0 < groups <= MAX_GROUPS and x_scales.shape == (r, kb) and offsets.shape == (groups + 1,) and
                weight_scales.shape == (groups, (out + 127) // BLOCK, kb) and offsets.is_contiguous() and
                (rows is None or rows.dtype is _I32 and rows.is_contiguous())):
            y = _empty_strided((n, out), (out, 1), output_dtype or _BF16)
            _check(_GROUPED(x.data_ptr(), xs, x_scales.data_ptr(), xss, r, None if rows is None else rows.data_ptr(), n, k,
                            weights.data_ptr(), wgs, ws, weight_scales.data_ptr(), wsgs, wss, out, groups,
                            offsets.data_ptr(), y.data_ptr(), out, t, _hip._raw_stream(index)), name)
            return y
    if rows is None:
        index = _device(name, x, x_scales, weights, weight_scales, offsets)
    else:
        index = _device(name, x, x_scales, weights, weight_scales, offsets, rows)
    if x.dim() != 2:
        raise ValueError(f"{name}: x must be [rows, K], not {list(x.shape)}")
    x, t, k, xs, x_scales, xss = _activations(name, x, x_scales)
    (groups, out, _), (wgs, ws, _), (wsgs, wss, _) = _weights(name, weights, weight_scales, k, 3)
    if groups > MAX_GROUPS:
        raise ValueError(f"{name}: at most {MAX_GROUPS} groups, not {groups}")
    if offsets.dtype is not _I32 or rows is not None and rows.dtype is not _I32:
        raise NotImplementedError(f"{name}: offsets and rows must be int32")
    if offsets.shape != (groups + 1,) or rows is not None and (rows.dim() != 1 or rows.shape[0] > MAX_ROWS):
        raise ValueError(f"{name}: offsets must be [{groups + 1}] and rows [R], not {list(offsets.shape)}"
                         f"{'' if rows is None else f' and {list(rows.shape)}'}")
    if not offsets.is_contiguous() or rows is not None and not rows.is_contiguous():
        raise NotImplementedError(f"{name}: offsets and rows must be contiguous")
    dtype, code = _out_type(name, output_dtype)
    n = t if rows is None else rows.shape[0]
    y = _matrix(x, n, out, dtype)
    if n:
        _call(index, "dsv2_grouped_linear_fp8_blocks", x.data_ptr(), xs, x_scales.data_ptr(), xss, t,
              None if rows is None else rows.data_ptr(), n, k, weights.data_ptr(), wgs, ws, weight_scales.data_ptr(), wsgs,
              wss, out, groups, offsets.data_ptr(), y.data_ptr(), out, code)
    return y
