"""The paged 4-bit latent cache without a GPU: what its functions and entry points refuse, before any
launch, and the plain implementations that the GPU tests hold it to."""

from __future__ import annotations

import ctypes
import os
import random
import shutil
import subprocess

import pytest
import torch

import paged_ref as R
from triton_kernels import _hip
from triton_kernels import paged_cache as P

BF = torch.bfloat16


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def good():
    """Arguments that each function takes, by function."""
    pages = torch.zeros(6, 16 * 400, dtype=torch.uint8)
    return {
        "paged_cache_step": [i32(6), i32(4), i32(4, 3), i32(6), 16, 9],
        "paged_slot_map": [i32(4), i32(4), i32(4, 3), 16, 9],
        "paged_cache_write_fp4": [torch.zeros(5, 576, dtype=BF), i32(5), pages],
        "paged_cache_read_fp4": [pages, i32(5), torch.zeros(5, 576, dtype=BF)],
        "attention_decode_paged_fp4": [torch.zeros(7, 16, 576, dtype=BF), pages, i32(4, 3), i32(4), 0.1, i32(5), 2,
                                       torch.zeros(7, 16, 512, dtype=BF)],
    }


@pytest.mark.parametrize("name", sorted(good()))
def test_functions_refuse_cpu_tensors(name):
    with pytest.raises(NotImplementedError, match="requires CUDA"):
        getattr(P, name)(*good()[name])


PAGES = lambda *shape: torch.zeros(*shape, dtype=torch.uint8)  # noqa: E731
REFUSED = [
    ("paged_cache_step", 0, i32(5), ValueError, "state must be"),
    ("paged_cache_step", 0, i32(6).long(), NotImplementedError, "state must be int32"),
    ("paged_cache_step", 1, i32(4, 1), ValueError, "delta must be"),
    ("paged_cache_step", 1, i32(8)[::2], NotImplementedError, "delta must be contiguous"),
    ("paged_cache_step", 2, i32(3, 3), ValueError, "block_table must be"),
    ("paged_cache_step", 2, i32(4, 0), ValueError, "block_table must be"),
    ("paged_cache_step", 2, i32(3, 4).T, NotImplementedError, "block_table rows"),
    ("paged_cache_step", 2, i32(1, 3).expand(4, 3), NotImplementedError, "block_table rows"),
    ("paged_cache_step", 2, i32(4, 3).float(), NotImplementedError, "block_table must be int32"),
    ("paged_cache_step", 3, i32(0), ValueError, "0 pages"),
    ("paged_cache_step", 4, 48, ValueError, "power of two"),
    ("paged_cache_step", 4, 2048, ValueError, "power of two"),
    ("paged_cache_step", 4, 0, ValueError, "power of two"),
    ("paged_cache_step", 5, -1, ValueError, "max_tokens"),
    ("paged_cache_step", 5, 2 ** 31, ValueError, "max_tokens"),
    ("paged_slot_map", 4, 2 ** 32 + 9, ValueError, "max_tokens"),
    ("paged_slot_map", 0, i32(3), ValueError, "counts must be"),
    ("paged_slot_map", 3, 12, ValueError, "power of two"),
    ("paged_slot_map", 4, -3, ValueError, "max_tokens"),
    ("paged_cache_write_fp4", 0, torch.zeros(5, 576), NotImplementedError, "rows must be bf16"),
    ("paged_cache_write_fp4", 0, torch.zeros(5, 512, dtype=BF), ValueError, "rows must be"),
    ("paged_cache_write_fp4", 0, torch.zeros(4, 576, dtype=BF), ValueError, "rows must be"),
    ("paged_cache_write_fp4", 0, torch.zeros(576, 5, dtype=BF).T, NotImplementedError, "contiguous rows"),
    ("paged_cache_write_fp4", 1, i32(5).long(), NotImplementedError, "slots must be int32"),
    ("paged_cache_write_fp4", 2, PAGES(6, 16 * 400 + 16), ValueError, "pages must be"),
    ("paged_cache_write_fp4", 2, PAGES(0, 400), ValueError, "pages must be"),
    ("paged_cache_write_fp4", 2, PAGES(6, 400).to(torch.int8), NotImplementedError, "pages must be uint8"),
    ("paged_cache_write_fp4", 2, PAGES(1, 400).expand(6, 400), NotImplementedError, "contiguous and apart"),
    ("paged_cache_read_fp4", 2, torch.zeros(5, 576), NotImplementedError, "out must be bf16"),
    ("paged_cache_read_fp4", 2, torch.zeros(1, 576, dtype=BF).expand(5, 576), NotImplementedError, "contiguous rows"),
    ("attention_decode_paged_fp4", 0, torch.zeros(7, 16, 576), NotImplementedError, "bf16 only"),
    ("attention_decode_paged_fp4", 0, torch.zeros(7, 16, 512, dtype=BF), ValueError, "expects q"),
    ("attention_decode_paged_fp4", 0, torch.zeros(7, 129, 576, dtype=BF), ValueError, "expects q"),
    ("attention_decode_paged_fp4", 0, torch.zeros(7, 576, 16, dtype=BF).transpose(1, 2), NotImplementedError,
     "contiguous last"),
    ("attention_decode_paged_fp4", 1, PAGES(6, 48 * 400), ValueError, "power of two"),
    ("attention_decode_paged_fp4", 2, i32(5, 3), ValueError, "block_table must be"),
    ("attention_decode_paged_fp4", 4, 0.0, ValueError, "softmax_scale must be positive"),
    ("attention_decode_paged_fp4", 4, -0.1, ValueError, "softmax_scale must be positive"),
    ("attention_decode_paged_fp4", 4, float("inf"), ValueError, "softmax_scale must be positive"),
    ("attention_decode_paged_fp4", 4, float("nan"), ValueError, "softmax_scale must be positive"),
    ("attention_decode_paged_fp4", 5, None, ValueError, "one query token a request"),
    ("attention_decode_paged_fp4", 5, i32(4), ValueError, "cu_q must be"),
    ("attention_decode_paged_fp4", 6, 0, ValueError, "max_q"),
    ("attention_decode_paged_fp4", 7, torch.zeros(7, 16, 576, dtype=BF), ValueError, "out must be"),
    ("attention_decode_paged_fp4", 7, torch.zeros(7, 1, 512, dtype=BF).expand(7, 16, 512), NotImplementedError,
     "rows must be contiguous"),
]


@pytest.mark.parametrize("name,at,value,error,text", REFUSED)
def test_functions_refuse_other_shapes_types_and_strides(monkeypatch, name, at, value, error, text):
    monkeypatch.setattr(P, "_device", lambda *a: 0)
    calls = []
    monkeypatch.setattr(P, "_call", lambda index, entry, *args: calls.append(entry))
    getattr(P, name)(*good()[name])
    assert len(calls) == 1
    args = good()[name]
    args[at] = value
    with pytest.raises(error, match=text):
        getattr(P, name)(*args)
    assert len(calls) == 1


@pytest.mark.parametrize("t,h", [(1, 1), (1, 5), (5, 1), (2, 2), (3, 4), (4, 3)])
def test_attention_refuses_outputs_whose_rows_overlap(monkeypatch, t, h):
    """Every pair of strides from a set, against all rows laid out."""
    monkeypatch.setattr(P, "_device", lambda *a: 0)
    calls = []
    monkeypatch.setattr(P, "_call", lambda index, entry, *args: calls.append(entry))
    q, pages, lens = torch.zeros(t, h, 576, dtype=BF), torch.zeros(6, 6400, dtype=torch.uint8), i32(t)
    strides = [8, 504, 512, 520, 768, 1016, 1024, 1032, 1536, 2048, 2552, 4096]
    for ts in strides:
        for hs in strides:
            at = sorted(i * ts + j * hs for i in range(t) for j in range(h))
            apart = all(y - x >= 512 for x, y in zip(at, at[1:]))
            out = torch.zeros(at[-1] + 512, dtype=BF).as_strided((t, h, 512), (ts, hs, 1))
            del calls[:]
            if apart:
                P.attention_decode_paged_fp4(q, pages, i32(t, 3), lens, 0.1, out=out)
            else:
                with pytest.raises(NotImplementedError, match="rows must be contiguous and apart"):
                    P.attention_decode_paged_fp4(q, pages, i32(t, 3), lens, 0.1, out=out)
            assert len(calls) == apart, (ts, hs)


@pytest.mark.parametrize("name", sorted(good()))
def test_functions_refuse_a_status_word_of_another_type_shape_or_device(monkeypatch, name):
    monkeypatch.setattr(P, "_device", lambda *a: -1)  # what get_device() says of a CPU tensor
    calls = []
    monkeypatch.setattr(P, "_call", lambda index, entry, word, *args: calls.append(word))
    word = i32(1)
    getattr(P, name)(*good()[name], status=word)
    getattr(P, name)(*good()[name])
    assert calls == [word.data_ptr(), None]
    for bad in (i32(2), i32(0), i32(1).long()):
        with pytest.raises(ValueError, match="status must be int32"):
            getattr(P, name)(*good()[name], status=bad)
    monkeypatch.setattr(P, "_device", lambda *a: 0)
    with pytest.raises(ValueError, match="status on cpu"):
        getattr(P, name)(*good()[name], status=word)
    with pytest.raises(ValueError, match="status on cpu"):
        P.check_paged_status(status=word)
    assert len(calls) == 2


def test_entry_points_refuse_bad_arguments_without_launching():
    one, odd = 1 << 20, (1 << 20) + 8  # never read: every call below is refused on the host

    def refused(match, entry, *args):
        with pytest.raises(_hip.HipKernelError, match=match):
            _hip.call(entry, *args, None, None)

    step = [one, one, 4, one, 3, 3, one, 6, 16, 9, odd << 4, one, one, one]
    for at, value, match in [(0, None, "null"), (2, 4097, "at most 4096"), (2, -1, "requests"), (4, 2, "block table"),
                             (5, 0, "block table"), (7, 0, "pages"), (7, 2 ** 28, "pages"), (8, 24, "power of two"),
                             (9, -1, "max_tokens"), (10, one + 8, "overlaps"), (11, None, "null")]:
        refused(match, "dsv2_paged_step", *step[:at], value, *step[at + 1:])
    slots = [one, one, 4, one, 3, 3, 16, 9, one, one, one]
    for at, value, match in [(1, None, "null"), (2, 5000, "at most"), (5, 2 ** 28, "block table"), (6, 0, "power of two")]:
        refused(match, "dsv2_paged_slots", *slots[:at], value, *slots[at + 1:])
    write = [one, 576, 5, one, one, 6400, 6, 16]
    for at, value, match in [(0, None, "null"), (0, odd, "alignment"), (1, 572, "bad shape"), (1, 580, "alignment"),
                             (2, -1, "bad shape"), (4, None, "null"), (4, odd, "alignment"), (5, 6384, "takes 6400"),
                             (5, 6408, "alignment"), (6, 0, "slots are int32"), (6, 2 ** 28, "slots are int32"),
                             (7, 17, "power of two")]:
        refused(match, "dsv2_paged_write_fp4", *write[:at], value, *write[at + 1:])
    read = [one, 6400, 6, 16, one, 5, one, 576]
    for at, value, match in [(4, None, "null"), (5, -1, "bad shape"), (6, odd, "alignment"), (7, 575, "bad shape")]:
        refused(match, "dsv2_paged_read_fp4", *read[:at], value, *read[at + 1:])
    size = _hip.lib.dsv2_mla_paged_workspace_size()
    attn = [one, 9216, 576, 7, 16, one, 6400, 6, 16, one, 3, 3, one, 4, one, 2, 0.1, one, 8192, 512, one, size]
    for at, value, match in [(0, None, "null"), (0, odd, "alignment"), (1, 9220, "alignment"), (3, -1, "bad shape"),
                             (4, 0, "bad shape"), (4, 129, "bad shape"), (8, 40, "power of two"), (10, 2, "block table"),
                             (11, 2 ** 28, "block table"), (12, None, "null"), (13, -1, "bad shape"), (13, 65536, "bad shape"),
                             (14, None, "bad shape"), (15, 0, "bad shape"),
                             (16, 0.0, "softmax_scale"), (16, -1.0, "softmax_scale"), (16, float("inf"), "softmax_scale"),
                             (16, float("nan"), "softmax_scale"), (18, 8196, "alignment"),
                             (20, None, "workspace"), (20, odd, "workspace"), (21, size - 1, "workspace")]:
        refused(match, "dsv2_mla_decode_paged_fp4", *attn[:at], value, *attn[at + 1:])


def test_attention_refuses_more_work_than_its_line_holds():
    one, size = 1 << 20, _hip.lib.dsv2_mla_paged_workspace_size()

    def refused(tokens, heads, requests, width, max_q):
        with pytest.raises(_hip.HipKernelError, match="groups of 16"):
            _hip.call("dsv2_mla_decode_paged_fp4", one, heads * 576, 576, tokens, heads, one, 6400, 6, 16, one, width,
                      width, one, requests, one, max_q, 0.1, one, heads * 512, 512, one, size, None, None)

    refused(65535, 128, 65535, 10000, 65535)
    refused(2 ** 20, 128, 1, 10000, 65535)     # one request's columns
    refused(2 ** 20, 16, 65535, 1000, 3000)    # all query tokens'
    refused(1, 1, 1, 2 ** 27 - 1, 1)           # a table past int32 tokens


def test_take_status_refuses_null_pointers():
    for args in ((None, 1 << 20), (1 << 20, None)):
        with pytest.raises(_hip.HipKernelError, match="paged_take_status: null"):
            _hip.call("dsv2_paged_take_status", *args, None)


def test_the_plain_block_format():
    """The reference of the GPU tests on values worked out by hand."""
    x = torch.zeros(4, 576)
    x[0, :4] = torch.tensor([6.0, 5.0, 2.5, -0.25])       # 6 is held: scale 1; ties 5 -> 4, 2.5 -> 2, 0.25 -> 0
    x[1, :4] = torch.tensor([6.03125, 1.75, 0.5, -3.5])   # past 6: scale 2: 3, 0.875 -> 1, 0.25 -> 0, 1.75 -> 2
    x[2, :3] = torch.tensor([float("inf"), 1.0, 2.0])
    x[3, 32:35] = torch.tensor([3.0e38, -3.3e38, 1.0e38])  # past 1.5 * 2^127: saturated at 6 * 2^125
    got = R.held(x.to(BF))
    assert got[0, :4].tolist() == [6.0, 4.0, 2.0, 0.0]
    assert got[1, :4].tolist() == [6.0, 2.0, 0.0, -4.0]
    assert got[2, :32].isnan().all() and not got[2, 32:].isnan().any()
    assert got[3, 32:34].tolist() == [6.0 * 2.0 ** 125, -6.0 * 2.0 ** 125]
    assert got[3, 34] == 2.0 * 2.0 ** 125  # 1e38 / 2^125 = 2.35


def test_the_plain_allocator_hands_out_and_takes_back():
    b = R.Allocator([2, 1], [[5, -1], [6, -1]], [9, 4, 7], 2, 1, 2)
    out, errors = b.step([1, -1], 3)
    # request 0 takes page 7 (ring position 2); request 1's page goes behind it, to position 0
    assert out == [[14, -1, -1], [2, -1, -1], [0, -1, -1]] and errors == 0
    assert b.ring == [6, 4, 7] and (b.head, b.count) == (0, 1) and b.lens == [3, 0]


def test_paged_latent_cache_shapes_and_refusals():
    from dsv2lite import PagedLatentCache

    c = PagedLatentCache(3, 5, max_len=100, n_pages=7, page_size=32, device="cpu")
    assert c.pages.shape == (3, 7, 32 * 400) and c.block_table.shape == (5, 4)
    assert c.state.tolist() == [0, 0, 0, 0, 0, 0, 7] and c.lens.data_ptr() == c.state.data_ptr()
    snap = c.snapshot()
    c.state.fill_(9)
    c.restore(snap)
    assert c.state.tolist() == [0, 0, 0, 0, 0, 0, 7] and c.free_tokens() == 224
    with pytest.raises(NotImplementedError, match="requires CUDA"):
        c.step(i32(5), 5)
    for kw, text in [(dict(page_size=48), "power of two"), (dict(page_size=2048), "power of two"),
                     (dict(requests=4097), "at most 4096"), (dict(n_pages=0), "positive"), (dict(max_len=0), "positive"),
                     (dict(n_pages=2 ** 26), "int32")]:
        with pytest.raises(ValueError, match=text):
            PagedLatentCache(**{**dict(n_layers=1, requests=2, max_len=10, n_pages=3, page_size=32, device="cpu"), **kw})


def test_step_refuses_other_query_starts(monkeypatch):
    monkeypatch.setattr(P, "_device", lambda *a: 0)
    calls = []
    monkeypatch.setattr(P, "_call", lambda index, entry, *args: calls.append(args[-1]))
    args, cu = good()["paged_cache_step"], i32(5)
    P.paged_cache_step(*args, cu_q=cu)
    P.paged_cache_step(*args)
    assert calls == [cu.data_ptr(), None]
    for bad, error in ((i32(4), ValueError), (i32(5).long(), NotImplementedError), (i32(10)[::2], NotImplementedError)):
        with pytest.raises(error, match="cu_q must be"):
            P.paged_cache_step(*args, cu_q=bad)
    assert len(calls) == 2


# --------------------------------------------------------------------------- the attention's line of items
ITEM_COST, WGS = 32, 256


@pytest.fixture(scope="module")
def line(tmp_path_factory):
    """csrc/paged_line.h, the arithmetic that the attention kernel cuts items with, in a host library."""
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host compiler")
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(P.__file__))), "csrc")
    where = tmp_path_factory.mktemp("line")
    src, lib = where / "line.cpp", where / "line.so"
    src.write_text('#include "paged_line.h"\n'
                   'extern "C" int cut_at(int t, int tiles) { return paged::cut_at(t, tiles); }\n'
                   'extern "C" void parts_of(int s, int n, int per, int wgs, int* out) {\n'
                   '  const paged::Parts p = paged::parts_of(s, n, per, wgs);\n'
                   '  out[0] = p.first;\n'
                   '  out[1] = p.last;\n'
                   '}\n')
    subprocess.run([cxx, "-std=c++17", "-O1", "-shared", "-fPIC", "-I", csrc, str(src), "-o", str(lib)], check=True)
    return ctypes.CDLL(str(lib))


def _parts(line, start, tiles, per, wgs):
    out = (ctypes.c_int * 2)()
    line.parts_of(start, tiles, per, wgs, out)
    return out[0], out[1]


def _grid(items, per):
    return min(WGS, max(1, sum(n + ITEM_COST for n in items)) // 16 + 1)


def _random_items(rng):
    return [rng.choice([rng.randint(1, 12), rng.randint(1, 40), rng.randint(1, 600), rng.randint(1, 12000)])
            for _ in range(rng.choice([1, 2, 7, 40, 300]))]


def test_every_tile_of_every_item_goes_to_one_piece_and_the_merge_knows_them(line):
    rng = random.Random(5)
    for _ in range(150):
        items = _random_items(rng)
        total = sum(n + ITEM_COST for n in items)
        per = max(-(-total // WGS), 16)
        wgs = _grid(items, per)
        start = 0
        for tiles in items:
            pieces = []
            for w in range(start // per, min(wgs, (start + tiles + ITEM_COST) // per + 1)):
                lo, hi = min(w * per, total), min((w + 1) * per, total)
                first, last = line.cut_at(lo - start, tiles), line.cut_at(hi - start, tiles)
                if first < last:
                    pieces.append((w, first, last))
            assert [p[1] for p in pieces] == [0] + [p[2] for p in pieces[:-1]] and pieces[-1][2] == tiles
            if len(pieces) > 1:
                assert min(p[2] - p[1] for p in pieces) >= 8
                assert [p[0] for p in pieces] == list(range(pieces[0][0], pieces[-1][0] + 1))
                assert _parts(line, start, tiles, per, wgs) == (pieces[0][0], pieces[-1][0])
            start += tiles + ITEM_COST


def test_an_item_that_grew_after_the_line_was_summed_is_joined_of_existing_parts(line):
    """A length that another stream changes while the attention runs may be read twice: the item's end then lies
    past the line, by a request's whole room at most."""
    rng = random.Random(6)
    found = 0
    for _ in range(3000):
        items = _random_items(rng)
        total = sum(n + ITEM_COST for n in items)
        per = max(-(-total // WGS), 16)
        wgs = _grid(items, per)
        w = rng.randrange(wgs)
        lo, hi = min(w * per, total), min((w + 1) * per, total)
        start = rng.randint(max(0, lo - rng.choice([20, 500, 100000])), lo)
        tiles = rng.choice([rng.randint(1, 100), rng.randint(1, 10 ** 6)])
        first, last = line.cut_at(lo - start, tiles), line.cut_at(hi - start, tiles)
        if lo < hi and 0 < first < last:  # this workgroup tells the merge of the item
            p0, p1 = _parts(line, start, tiles, per, wgs)
            assert 0 <= p0 < w <= p1 < wgs, (items, start, tiles, w)
            found += 1
    assert found > 500
