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
skip what they concern and are reported by ``check_paged_status``; attention takes table entries that
name no page for tokens of zeros.  Lengths are held to what the table has room for, a negative one to
zero, without a report.  Errors are kept in ``status``, an int32 [1] tensor of zeros on the same GPU
that the callers who share it pass to each call; without one the calls of a device share a word of the
module's, whose first use has to be outside graph capture.
"""

from __future__ import annotations

import torch

from . import _hip

LAT, ROPE = 512, 64
ROW = LAT + ROPE
TOKEN_BYTES = LAT // 2 + 2 * ROPE + LAT // 32  # 400
MAX_REQUESTS = 4096
MAX_HEADS = 128
MAX_TOKENS = 2 ** 31 - 1

# These calls launch kernels of 2 to 10 us, so their own host time is looked at: a launch takes 3 us of it, a
# torch.empty 1.3, an attribute of a tensor 0.05 to 0.1.
_BF16, _I32, _U8 = torch.bfloat16, torch.int32, torch.uint8
_PAGE_SIZES = frozenset(1 << i for i in range(11))
_ENTRY = {n: getattr(_hip.lib, n) for n in ("dsv2_paged_step_queries", "dsv2_paged_slots", "dsv2_paged_write_fp4",
                                            "dsv2_paged_read_fp4", "dsv2_mla_decode_paged_fp4", "dsv2_paged_take_status")}
_WORKSPACE = _hip.lib.dsv2_mla_paged_workspace_size()  # bytes
_STATUS: dict = {}  # device index -> (int32 [1] status word of the functions below, its address)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _status(index: int) -> tuple[torch.Tensor, int]:
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("paged cache: the first call on a device must be outside graph capture")
    st = torch.zeros(1, dtype=_I32, device=torch.device("cuda", index))
    torch.cuda.current_stream(index).synchronize()  # other streams' calls find it cleared
    return _STATUS.setdefault(index, (st, st.data_ptr()))


def check_paged_status(device: torch.device | str = "cuda", status: torch.Tensor | None = None) -> None:
    """Raise if a call with this ``status`` (without one: a call on `device` without one) has skipped something since
    the last check.  Waits for all streams of the device, on any of which such a call may be."""
    name = "check_paged_status"
    if status is None:
        index = torch.device(device).index
        index = torch.cuda.current_device() if index is None else index
        known = _STATUS.get(index)
        if known is None:
            return
        status = known[0]
    index = _device(name, status)
    at = _word(name, status, index)
    torch.cuda.synchronize(index)
    # read and cleared at once: what another thread's call finds meanwhile is left for the next check
    taken = torch.empty_like(status)
    _call(index, "dsv2_paged_take_status", at, taken.data_ptr())
    bits = int(taken.item())
    if not bits:
        return
    what = [text for bit, text in ((1, "a request outgrew its block table"), (2, "no free page was left"),
                                   (4, "a slot, page or position lay outside the pool or block table"),
                                   (8, "there were more new tokens than max_tokens or max_q")) if bits & bit]
    raise RuntimeError("paged cache: " + "; ".join(what) + "; those tokens were skipped")


def _word(name: str, status: torch.Tensor, index: int) -> int:
    """The address of a call's own status word."""
    if status.dtype is not _I32 or status.numel() != 1:
        raise ValueError(f"{name}: status must be int32 [1], not {status.dtype} {list(status.shape)}")
    if status.get_device() != index:
        raise ValueError(f"{name}: status on {status.device}")
    return status.data_ptr()


def _call(index: int, entry: str, word: int | None, *args) -> None:
    """The entry point on the device's current stream, with the device as the current one; `word`: the address of the
    call's status word, None for the device's."""
    if _current_device() != index:
        with torch.cuda.device(index):
            return _call(index, entry, word, *args)
    if word is None:
        word = (_STATUS.get(index) or _status(index))[1]
    rc = _ENTRY[entry](*args, word, _hip._raw_stream(index))
    if rc:
        raise _hip.HipKernelError(f"{entry} failed (status {rc}): "
                                  f"{_hip.lib.dsv2_last_error_message().decode(errors='replace')}")


def _device(name: str, *ts: torch.Tensor) -> int:
    """The index of the one GPU that all tensors are on."""
    index = ts[0].get_device()
    for t in ts:
        if t.get_device() != index or index < 0:
            if not t.is_cuda:
                raise NotImplementedError(f"{name} requires CUDA (HIP) tensors")
            raise ValueError(f"{name}: tensors on {ts[0].device} and {t.device}")
    return index


def _int32(name: str, what: str, t: torch.Tensor, n: int | None = None) -> int:
    """The length of an int32 vector (n, if given)."""
    if t.dtype is not _I32:
        raise NotImplementedError(f"{name}: {what} must be int32")
    shape = t.shape
    if len(shape) != 1 or (n is not None and shape[0] != n):
        raise ValueError(f"{name}: {what} must be [{'n' if n is None else n}], not {list(shape)}")
    if not t.is_contiguous():
        raise NotImplementedError(f"{name}: {what} must be contiguous")
    return shape[0]


def _table(name: str, t: torch.Tensor, n: int) -> tuple[int, int]:
    """(row stride, width) of a block table."""
    if t.dtype is not _I32:
        raise NotImplementedError(f"{name}: block_table must be int32")
    shape = t.shape
    if len(shape) != 2 or shape[0] != n or shape[1] == 0:
        raise ValueError(f"{name}: block_table must be [{n}, pages of a request], not {list(shape)}")
    width = shape[1]
    rs, cs = t.stride()
    if cs != 1 and width > 1 or rs < width and n > 1:
        raise NotImplementedError(f"{name}: block_table rows must be contiguous and apart")
    return (rs if rs > width else width), width


def _pool(name: str, pages: torch.Tensor) -> tuple[int, int, int]:
    """(page stride in bytes, pages, page size) of a pool."""
    if pages.dtype is not _U8:
        raise NotImplementedError(f"{name}: pages must be uint8")
    shape = pages.shape
    if len(shape) != 2 or shape[0] == 0 or shape[1] == 0 or shape[1] % TOKEN_BYTES:
        raise ValueError(f"{name}: pages must be [n_pages, page_size * {TOKEN_BYTES}], not {list(shape)}")
    n, width = shape
    stride, cs = pages.stride()
    if cs != 1 or stride < width and n > 1:
        raise NotImplementedError(f"{name}: pages must be contiguous and apart")
    page_size = width // TOKEN_BYTES
    _page_size(name, page_size)
    return (stride if stride > width else width), n, page_size


def _page_size(name: str, page_size: int) -> None:
    if page_size not in _PAGE_SIZES:
        raise ValueError(f"{name}: page_size must be a power of two up to 1024, not {page_size}")


def paged_cache_step(state: torch.Tensor, delta: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                     page_size: int, max_tokens: int, status: torch.Tensor | None = None,
                     cu_q: torch.Tensor | None = None) -> tuple[torch.Tensor, ...]:
    """One step of the requests' lengths; returns (state after the step, slots, positions, rows).

    ``state`` int32 [B + 2]: the B lengths, then head and count of the ring ``free_pages`` (int32
    [n_pages]; its free page numbers are free_pages[(head + i) % n_pages] for i < count).
    ``delta`` int32 [B]: tokens that each request gains (> 0) or drops from its end (< 0; at most
    all).  Growing requests take the ring's next pages into their ``block_table`` [B, width] rows,
    shrinking ones put the pages they empty behind the free ones (handed out from the next step
    on); both tensors change in place, in places that the step does not read, so the call repeated
    on the same ``state`` does the same.  New token i, requests in order, has slots[i],
    positions[i] and rows[i] (its request); entries from the last new token to ``max_tokens`` are
    -1.  A request whose tokens do not fit the table, ``max_tokens`` or the free pages keeps its
    length; its tokens get -1 and check_paged_status raises.  Both are counted in the requests' order, what
    was refused with the rest: behind a request refused for tokens all that grow are refused, behind one
    refused for pages all that need a page.  One that would outgrow the table counts its tokens, no pages.

    ``cu_q`` int32 [B + 1], if given, receives where each request's new tokens begin and the last one's end,
    refused ones' among them: ``attention_decode_paged_fp4``'s argument for a query of each new token."""
    name = "paged_cache_step"
    index = _device(name, state, delta, block_table, free_pages)
    n = _int32(name, "delta", delta)
    _int32(name, "state", state, n + 2)
    pages = _int32(name, "free_pages", free_pages)
    _page_size(name, page_size)
    ts, width = _table(name, block_table, n)
    if n > MAX_REQUESTS or pages == 0 or not 0 <= max_tokens <= MAX_TOKENS:
        raise ValueError(f"{name}: {n} requests (at most {MAX_REQUESTS}), {pages} pages, max_tokens {max_tokens}")
    cu = None
    if cu_q is not None:
        _device(name, state, cu_q)
        _int32(name, "cu_q", cu_q, n + 1)
        cu = cu_q.data_ptr()
    outs = state.new_empty(n + 2 + 3 * max_tokens)  # one allocation: the state, then the three maps
    if n == 0:
        outs.fill_(-1)[:2] = state
        if cu is not None:
            cu_q.zero_()
    else:
        at = outs.data_ptr()
        maps, size = at + 4 * n + 8, 4 * max_tokens
        _call(index, "dsv2_paged_step_queries", None if status is None else _word(name, status, index),
              state.data_ptr(), delta.data_ptr(), n, block_table.data_ptr(), ts, width, free_pages.data_ptr(), pages,
              page_size, max_tokens, at, maps, maps + size, maps + 2 * size, cu)
    return torch.unsafe_split_with_sizes(outs, (n + 2, max_tokens, max_tokens, max_tokens))


def paged_slot_map(starts: torch.Tensor, counts: torch.Tensor, block_table: torch.Tensor, page_size: int,
                   max_tokens: int,
                   status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(slots, positions, rows) of the tokens [starts[b], starts[b] + counts[b]) of every request, one
    after the other, int32 [max_tokens]; -1 from the last one on, and for positions or pages out of
    range."""
    name = "paged_slot_map"
    index = _device(name, starts, counts, block_table)
    n = _int32(name, "starts", starts)
    _int32(name, "counts", counts, n)
    _page_size(name, page_size)
    ts, width = _table(name, block_table, n)
    if n > MAX_REQUESTS or not 0 <= max_tokens <= MAX_TOKENS:
        raise ValueError(f"{name}: {n} requests (at most {MAX_REQUESTS}), max_tokens {max_tokens}")
    maps = starts.new_empty(3 * max_tokens)
    if n == 0 or max_tokens == 0:
        maps.fill_(-1)
    else:
        at, size = maps.data_ptr(), 4 * max_tokens
        _call(index, "dsv2_paged_slots", None if status is None else _word(name, status, index), starts.data_ptr(),
              counts.data_ptr(), n, block_table.data_ptr(), ts, width, page_size, max_tokens, at, at + size, at + 2 * size)
    return torch.unsafe_split_with_sizes(maps, (max_tokens, max_tokens, max_tokens))


def _cache_rows(name: str, what: str, rows: torch.Tensor, n: int) -> int:
    """Row stride of [n, 576] bf16 cache rows; 0 for one row that is read for all."""
    if rows.dtype is not _BF16:
        raise NotImplementedError(f"{name}: {what} must be bf16")
    if rows.shape != (n, ROW):
        raise ValueError(f"{name}: {what} must be [{n}, {ROW}], not {list(rows.shape)}")
    rs, cs = rows.stride()
    if cs != 1 or rs < ROW and n > 1 and (rs or what == "out"):
        raise NotImplementedError(f"{name}: {what} must have contiguous rows")
    return rs if n > 1 else ROW


def paged_cache_write_fp4(rows: torch.Tensor, slots: torch.Tensor, pages: torch.Tensor,
                          status: torch.Tensor | None = None) -> None:
    """Round cache rows (bf16 [n, 576]: normalised latent | rotated key, a row stride that is a
    multiple of 8, or 0 for one row) into ``slots`` (int32 [n]) of ``pages``; a row with a negative slot is left out.
    Rows with the same slot have to be the same: of different ones a mixture may stay."""
    name = "paged_cache_write_fp4"
    index = _device(name, rows, slots, pages)
    n = _int32(name, "slots", slots)
    rs = _cache_rows(name, "rows", rows, n)
    page_stride, n_pages, page_size = _pool(name, pages)
    if n:
        _call(index, "dsv2_paged_write_fp4", None if status is None else _word(name, status, index), rows.data_ptr(),
              rs, n, slots.data_ptr(), pages.data_ptr(), page_stride, n_pages, page_size)


def paged_cache_read_fp4(pages: torch.Tensor, slots: torch.Tensor, out: torch.Tensor | None = None,
                         status: torch.Tensor | None = None) -> torch.Tensor:
    """The bf16 rows [n, 576] that ``slots`` (int32 [n]) hold, exactly; zeros for a negative slot."""
    name = "paged_cache_read_fp4"
    index = _device(name, pages, slots)
    n = _int32(name, "slots", slots)
    page_stride, n_pages, page_size = _pool(name, pages)
    if out is None:
        out, os = torch.empty((n, ROW), dtype=_BF16, device=slots.device), ROW
    else:
        _device(name, pages, out)
        os = _cache_rows(name, "out", out, n)
    if n:
        _call(index, "dsv2_paged_read_fp4", None if status is None else _word(name, status, index), pages.data_ptr(),
              page_stride, n_pages, page_size, slots.data_ptr(), n, out.data_ptr(), os)
    return out


def _rows_apart(t: int, ts: int, h: int, hs: int) -> bool:
    """No two of the t * h rows of 512 values, ts and hs apart, have a value in common."""
    if h <= 1 or t <= 1:
        return (h <= 1 or hs >= LAT) and (t <= 1 or ts >= LAT)
    if min(ts, hs) < LAT:
        return False
    if ts >= (h - 1) * hs + LAT or hs >= (t - 1) * ts + LAT:  # one within the other
        return True
    # else the tokens next to every head's offset
    return all(abs(j * hs - i * ts) >= LAT for j in range(1, h) for i in (j * hs // ts, j * hs // ts + 1) if i < t)


def attention_decode_paged_fp4(q: torch.Tensor, pages: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
                               softmax_scale: float, cu_q: torch.Tensor | None = None, max_q: int = 1,
                               out: torch.Tensor | None = None,
                               status: torch.Tensor | None = None) -> torch.Tensor:
    """Absorbed-MLA attention over the pages: q [T, H, 576] bf16 (q_nope W_UK | rotated q_pe) -> the
    latent outputs [T, H, 512] bf16 that W_UV takes, fp32 softmax over each request's ``lens[b]``
    cached tokens.

    Without ``cu_q`` query token b belongs to request b.  With it (int32 [B + 1], ascending) request
    b owns query tokens cu_q[b] .. cu_q[b + 1], at most ``max_q`` of them, and they are its last
    cached tokens: the last one sees all, each one before it a token less.  Where ``cu_q``'s tokens are a
    step's new ones, a request that does not grow has none, so rows are not the requests' numbers
    (``paged_cache_step`` forms it).  A query that sees nothing
    gives zeros; query tokens past cu_q[B] are not written (in a fresh ``out`` they are undefined).
    Sums are fp32 with weights up to 2^8, so latents past some 2^100 may overflow to infinity.
    Up to 128 heads; q and out may have any token and head strides that are multiples of 8 (out's rows apart).
    Up to 65,535 requests and ``max_q``; (T * H / 16 + B) * (table width * page size / 16 + 32) up to 2^30."""
    name = "attention_decode_paged_fp4"
    index = _device(name, q, pages, block_table, lens)
    if q.dtype is not _BF16:
        raise NotImplementedError(f"{name} supports bf16 only")
    shape = q.shape
    if len(shape) != 3 or shape[2] != ROW or not 0 < shape[1] <= MAX_HEADS:
        raise ValueError(f"{name} expects q [tokens, heads up to {MAX_HEADS}, {ROW}], not {list(shape)}")
    t, h, _ = shape
    n = _int32(name, "lens", lens)
    page_stride, n_pages, page_size = _pool(name, pages)
    ts, width = _table(name, block_table, n)
    if cu_q is None:
        if n != t or max_q != 1:
            raise ValueError(f"{name}: without cu_q there is one query token a request ({t} for {n})")
        cu = None
    else:
        _device(name, q, cu_q)
        _int32(name, "cu_q", cu_q, n + 1)
        if max_q < 1:
            raise ValueError(f"{name}: max_q must be positive")
        max_q, cu = min(max_q, max(t, 1)), cu_q.data_ptr()
    if not 0.0 < softmax_scale <= 1e30:
        raise ValueError(f"{name}: softmax_scale must be positive and finite, not {softmax_scale}")
    q_ts, q_hs, q_ds = q.stride()
    if q_ds != 1:
        raise NotImplementedError(f"{name} needs a contiguous last dimension")
    if t == 1:  # strides that are never taken may be anything
        q_ts = 0
    if h == 1:
        q_hs = 0
    if out is None:
        out = q.new_empty((t, h, LAT))
        o_ts, o_hs = h * LAT, LAT
    else:
        _device(name, q, out)
        if out.dtype is not _BF16:
            raise NotImplementedError(f"{name} writes bf16 only")
        if out.shape != (t, h, LAT):
            raise ValueError(f"{name}: out must be [{t}, {h}, {LAT}], not {list(out.shape)}")
        o_ts, o_hs, o_ds = out.stride()
        if o_ds != 1 or not _rows_apart(t, o_ts, h, o_hs):
            raise NotImplementedError(f"{name}: out's rows must be contiguous and apart")
        if t == 1:
            o_ts = 0
        if h == 1:
            o_hs = 0
    if t == 0 or n == 0:
        return out
    ws = pages.new_empty(_WORKSPACE)
    _call(index, "dsv2_mla_decode_paged_fp4", None if status is None else _word(name, status, index), q.data_ptr(), q_ts,
          q_hs, t, h, pages.data_ptr(), page_stride, n_pages, page_size, block_table.data_ptr(), ts, width, lens.data_ptr(),
          n, cu, max_q, softmax_scale, out.data_ptr(), o_ts, o_hs, ws.data_ptr(), _WORKSPACE)
    return out
