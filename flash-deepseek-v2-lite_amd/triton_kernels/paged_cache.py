"""Paged latent cache held in 4 bits: block tables and slot maps on the GPU, rows into pages and
back, absorbed-MLA decode attention over the pages.

No counterpart in the reference, whose cache is one expanded bf16 tensor of fixed length
(src/run.py:81-99); these stand beside ``attention_decode_batch`` for callers whose requests share
one pool of memory.

One layer's pool is ``pages`` [n_pages, page_size * 400] uint8 (any stride between pages that is a
multiple of 16).  A token takes 400 bytes: its 512 latent values as e2m1 codes in blocks of 32 with
one power-of-two scale each (``include/dsv2lite.h`` has the layout), its 64 rotary keys in bf16.
Slot ``p * page_size + i`` names token i of page p.  Token t of request b lies in page
``block_table[b, t // page_size]``; one table serves all layers.

Errors that only the device can see (no free page, a full block table, a slot outside the pool)
skip what they concern and are reported by ``check_paged_status``.
"""

from __future__ import annotations

import torch

from . import _hip
from ._checks import require_cuda

LAT, ROPE = 512, 64
ROW = LAT + ROPE
TOKEN_BYTES = LAT // 2 + 2 * ROPE + LAT // 32  # 400
MAX_REQUESTS = 4096
MAX_HEADS = 128

_BF16, _I32, _U8 = torch.bfloat16, torch.int32, torch.uint8
_STATUS: dict = {}  # device index -> int32 [1] status word of the functions below


def _status(dev: torch.device) -> torch.Tensor:
    st = _STATUS.get(dev.index)
    if st is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("paged cache: the first call on a device must be outside graph capture")
        st = _STATUS[dev.index] = torch.zeros(1, dtype=_I32, device=dev)
        torch.cuda.current_stream(dev).synchronize()  # other streams' calls find it cleared
    return st


def check_paged_status(device: torch.device | str = "cuda") -> None:
    """Raise if a call on `device` since the last check skipped something (synchronises)."""
    dev = torch.device(device)
    st = _STATUS.get(torch.cuda.current_device() if dev.index is None else dev.index)
    bits = 0 if st is None else int(st.item())
    if not bits:
        return
    st.zero_()
    what = [text for bit, text in ((1, "a request outgrew its block table"), (2, "no free page was left"),
                                   (4, "a slot, page or position lay outside the pool or block table"),
                                   (8, "there were more new tokens than max_tokens or max_q")) if bits & bit]
    raise RuntimeError("paged cache: " + "; ".join(what) + "; those tokens were skipped")


def _call(dev: torch.device, name: str, *args) -> None:
    """The entry point on dev's current stream, with dev as the current device."""
    if torch.cuda.current_device() == dev.index:
        _hip.call(name, *args, _status(dev).data_ptr(), _hip.stream_ptr(dev))
        return
    with torch.cuda.device(dev):
        _hip.call(name, *args, _status(dev).data_ptr(), _hip.stream_ptr(dev))


def _same_device(name: str, *ts: torch.Tensor) -> torch.device:
    require_cuda(name, *ts)
    dev = ts[0].device
    for t in ts[1:]:
        if t.device != dev:
            raise ValueError(f"{name}: tensors on {dev} and {t.device}")
    return dev


def _int32(name: str, what: str, t: torch.Tensor, n: int | None = None) -> None:
    if t.dtype != _I32:
        raise NotImplementedError(f"{name}: {what} must be int32")
    if t.ndim != 1 or (n is not None and t.shape[0] != n):
        raise ValueError(f"{name}: {what} must be [{'n' if n is None else n}]")
    if t.shape[0] > 1 and t.stride(0) != 1:
        raise NotImplementedError(f"{name}: {what} must be contiguous")


def _table(name: str, t: torch.Tensor, n: int) -> tuple[int, int]:
    """(row stride, width) of a block table."""
    if t.dtype != _I32:
        raise NotImplementedError(f"{name}: block_table must be int32")
    if t.ndim != 2 or t.shape[0] != n or t.shape[1] == 0:
        raise ValueError(f"{name}: block_table must be [{n}, pages of a request]")
    rs, cs = t.stride()
    width = t.shape[1]
    if cs != 1 and width > 1 or rs < width and n > 1:
        raise NotImplementedError(f"{name}: block_table rows must be contiguous and apart")
    return max(rs, width), width


def _pool(name: str, pages: torch.Tensor) -> tuple[int, int, int]:
    """(page stride in bytes, pages, page size) of a pool."""
    if pages.dtype != _U8:
        raise NotImplementedError(f"{name}: pages must be uint8")
    if pages.ndim != 2 or pages.shape[0] == 0 or pages.shape[1] == 0 or pages.shape[1] % TOKEN_BYTES:
        raise ValueError(f"{name}: pages must be [n_pages, page_size * {TOKEN_BYTES}]")
    n, width = pages.shape
    ps, cs = pages.stride()
    if cs != 1 or ps < width and n > 1:
        raise NotImplementedError(f"{name}: pages must be contiguous and apart")
    return max(ps, width), n, width // TOKEN_BYTES


def _page_size(name: str, page_size: int) -> None:
    if page_size < 1 or page_size > 1024 or page_size & (page_size - 1):
        raise ValueError(f"{name}: page_size must be a power of two up to 1024, not {page_size}")


def paged_cache_step(state: torch.Tensor, delta: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                     page_size: int, max_tokens: int) -> tuple[torch.Tensor, ...]:
    """One step of the requests' lengths; returns (state after the step, slots, positions, rows).

    ``state`` int32 [B + 2]: the B lengths, then head and count of the ring ``free_pages`` (int32
    [n_pages]; its free page numbers are free_pages[(head + i) % n_pages] for i < count).
    ``delta`` int32 [B]: tokens that each request gains (> 0) or drops from its end (< 0; at most
    all).  Growing requests take the ring's next pages into their ``block_table`` [B, width] rows,
    shrinking ones put the pages they empty behind the free ones (handed out from the next step
    on); both tensors change in place, in places that the step does not read, so the call repeated
    on the same ``state`` does the same.  New token i, requests in order, has slots[i],
    positions[i] and rows[i] (its request); entries from the last new token to ``max_tokens`` are
    -1.  A request whose tokens do not fit the table, ``max_tokens`` or the free pages that the
    requests before it leave keeps its length; its tokens get -1 and check_paged_status raises."""
    name = "paged_cache_step"
    dev = _same_device(name, state, delta, block_table, free_pages)
    n = delta.shape[0] if delta.ndim == 1 else -1
    _int32(name, "delta", delta)
    _int32(name, "state", state, n + 2)
    _int32(name, "free_pages", free_pages)
    _page_size(name, page_size)
    ts, width = _table(name, block_table, n)
    if n > MAX_REQUESTS or free_pages.shape[0] == 0 or max_tokens < 0:
        raise ValueError(f"{name}: {n} requests (at most {MAX_REQUESTS}), {free_pages.shape[0]} pages, max_tokens "
                         f"{max_tokens}")
    after = torch.empty(n + 2, dtype=_I32, device=dev)
    maps = torch.empty((3, max_tokens), dtype=_I32, device=dev)
    if n == 0:
        return after.copy_(state), *maps.fill_(-1).unbind(0)
    at = maps.data_ptr()
    _call(dev, "dsv2_paged_step", state.data_ptr(), delta.data_ptr(), n, block_table.data_ptr(), ts, width,
          free_pages.data_ptr(), free_pages.shape[0], page_size, max_tokens, after.data_ptr(), at,
          at + 4 * max_tokens, at + 8 * max_tokens)
    return after, *maps.unbind(0)


def paged_slot_map(starts: torch.Tensor, counts: torch.Tensor, block_table: torch.Tensor, page_size: int,
                   max_tokens: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(slots, positions, rows) of the tokens [starts[b], starts[b] + counts[b]) of every request, one
    after the other, int32 [max_tokens]; -1 from the last one on, and for positions or pages out of
    range."""
    name = "paged_slot_map"
    dev = _same_device(name, starts, counts, block_table)
    n = starts.shape[0] if starts.ndim == 1 else -1
    _int32(name, "starts", starts)
    _int32(name, "counts", counts, n)
    _page_size(name, page_size)
    ts, width = _table(name, block_table, n)
    if n > MAX_REQUESTS or max_tokens < 0:
        raise ValueError(f"{name}: {n} requests (at most {MAX_REQUESTS}), max_tokens {max_tokens}")
    maps = torch.empty((3, max_tokens), dtype=_I32, device=dev)
    if n == 0 or max_tokens == 0:
        return maps.fill_(-1).unbind(0)
    at = maps.data_ptr()
    _call(dev, "dsv2_paged_slots", starts.data_ptr(), counts.data_ptr(), n, block_table.data_ptr(), ts, width,
          page_size, max_tokens, at, at + 4 * max_tokens, at + 8 * max_tokens)
    return maps.unbind(0)


def _cache_rows(name: str, what: str, rows: torch.Tensor, n: int) -> int:
    """Row stride of [n, 576] bf16 cache rows."""
    if rows.dtype != _BF16:
        raise NotImplementedError(f"{name}: {what} must be bf16")
    if rows.shape != (n, ROW):
        raise ValueError(f"{name}: {what} must be [{n}, {ROW}]")
    rs, cs = rows.stride()
    if cs != 1 or rs < ROW and n > 1:
        raise NotImplementedError(f"{name}: {what} must have contiguous rows")
    return max(rs, ROW)


def paged_cache_write_fp4(rows: torch.Tensor, slots: torch.Tensor, pages: torch.Tensor) -> None:
    """Round cache rows (bf16 [n, 576]: normalised latent | rotated key, any row stride that is a
    multiple of 8) into ``slots`` (int32 [n]) of ``pages``; a row with a negative slot is left out.
    Of two rows with the same slot either may stay."""
    name = "paged_cache_write_fp4"
    dev = _same_device(name, rows, slots, pages)
    _int32(name, "slots", slots)
    n = slots.shape[0]
    rs = _cache_rows(name, "rows", rows, n)
    page_stride, n_pages, page_size = _pool(name, pages)
    if n:
        _call(dev, "dsv2_paged_write_fp4", rows.data_ptr(), rs, n, slots.data_ptr(), pages.data_ptr(), page_stride,
              n_pages, page_size)


def paged_cache_read_fp4(pages: torch.Tensor, slots: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """The bf16 rows [n, 576] that ``slots`` (int32 [n]) hold, exactly; zeros for a negative slot."""
    name = "paged_cache_read_fp4"
    dev = _same_device(name, pages, slots) if out is None else _same_device(name, pages, slots, out)
    _int32(name, "slots", slots)
    n = slots.shape[0]
    page_stride, n_pages, page_size = _pool(name, pages)
    if out is None:
        out, os = torch.empty((n, ROW), dtype=_BF16, device=dev), ROW
    else:
        os = _cache_rows(name, "out", out, n)
    if n:
        _call(dev, "dsv2_paged_read_fp4", pages.data_ptr(), page_stride, n_pages, page_size, slots.data_ptr(), n,
              out.data_ptr(), os)
    return out


def attention_decode_paged_fp4(q: torch.Tensor, pages: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
                               softmax_scale: float, cu_q: torch.Tensor | None = None, max_q: int = 1,
                               out: torch.Tensor | None = None) -> torch.Tensor:
    """Absorbed-MLA attention over the pages: q [T, H, 576] bf16 (q_nope W_UK | rotated q_pe) -> the
    latent outputs [T, H, 512] bf16 that W_UV takes, fp32 softmax over each request's ``lens[b]``
    cached tokens.

    Without ``cu_q`` query token b belongs to request b.  With it (int32 [B + 1], ascending) request
    b owns query tokens cu_q[b] .. cu_q[b + 1], at most ``max_q`` of them, and they are its last
    cached tokens: the last one sees all, each one before it a token less.  A query that sees nothing
    gives zeros; query tokens past cu_q[B] are not written (in a fresh ``out`` they are undefined).
    Up to 128 heads; q and out may have any token and head strides that are multiples of 8."""
    name = "attention_decode_paged_fp4"
    dev = _same_device(name, q, pages, block_table, lens)
    if q.dtype != _BF16:
        raise NotImplementedError(f"{name} supports bf16 only")
    if q.ndim != 3 or q.shape[2] != ROW or not 0 < q.shape[1] <= MAX_HEADS:
        raise ValueError(f"{name} expects q [tokens, heads up to {MAX_HEADS}, {ROW}]")
    t, h, _ = q.shape
    _int32(name, "lens", lens)
    n = lens.shape[0]
    page_stride, n_pages, page_size = _pool(name, pages)
    _page_size(name, page_size)
    ts, width = _table(name, block_table, n)
    if cu_q is None:
        if n != t or max_q != 1:
            raise ValueError(f"{name}: without cu_q there is one query token a request ({t} for {n})")
    else:
        _same_device(name, q, cu_q)
        _int32(name, "cu_q", cu_q, n + 1)
        if max_q < 1:
            raise ValueError(f"{name}: max_q must be positive")
        max_q = min(max_q, max(t, 1))
    q_ts, q_hs, q_ds = q.stride()
    if q_ds != 1:
        raise NotImplementedError(f"{name} needs a contiguous last dimension")
    if out is None:
        out = torch.empty((t, h, LAT), dtype=_BF16, device=dev)
        o_ts, o_hs = h * LAT, LAT
    else:
        _same_device(name, q, out)
        if out.dtype != _BF16:
            raise NotImplementedError(f"{name} writes bf16 only")
        if out.shape != (t, h, LAT):
            raise ValueError(f"{name}: out must be [{t}, {h}, {LAT}]")
        o_ts, o_hs, o_ds = out.stride()
        if o_ds != 1 or h > 1 and o_hs < LAT or t > 1 and o_ts < LAT:
            raise NotImplementedError(f"{name}: out's rows must be contiguous and apart")
    if t == 0 or n == 0:
        return out
    size = _hip.lib.dsv2_mla_paged_workspace_size(n, max_q, h)
    ws = torch.empty(size, dtype=_U8, device=dev)
    _call(dev, "dsv2_mla_decode_paged_fp4", q.data_ptr(), q_ts, q_hs, t, h, pages.data_ptr(), page_stride, n_pages,
          page_size, block_table.data_ptr(), ts, width, lens.data_ptr(), n, None if cu_q is None else cu_q.data_ptr(),
          max_q, float(softmax_scale), out.data_ptr(), o_ts, o_hs, ws.data_ptr(), size)
    return out
