"""The paged 4-bit latent cache on the GPU against plain implementations in 64 bits: block tables and
slot maps exactly, the block format exactly (every bf16 value), attention within the bound that its
roundings give, and the operators together as a serving loop uses them."""

from __future__ import annotations

import random

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from triton_kernels import _hip
    from triton_kernels import paged_cache as P

import paged_ref as R

DEV = "cuda"
BF = torch.bfloat16
SCALE = 0.1147


@pytest.fixture(autouse=True)
def no_error_bits_left():
    """No call but those that are meant to sets a device status bit."""
    yield
    P.check_paged_status()


def rnd(*shape, seed=0, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(BF)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def pool(n_pages, ps, fill=None):
    """A pool of pages: every byte `fill`, or rows of normal values."""
    pages = torch.full((n_pages, ps * R.TOKEN), 255 if fill is None else fill, dtype=torch.uint8, device=DEV)
    if fill is None:
        P.paged_cache_write_fp4(rnd(n_pages * ps, R.ROW, seed=n_pages), torch.arange(n_pages * ps, device=DEV).int(),
                                pages)
    return pages


def batch(lens, ps, seed=0, spare=3, fill=None):
    """(pages, table, the requests' rows in 64 bits): pages dealt out in random order; what no request
    owns, the unused ends of their last pages included, is bytes 255 (NaN scales and keys)."""
    rng = random.Random(seed)
    need = [-(-n // ps) for n in lens]
    order = list(range(sum(need) + spare))
    rng.shuffle(order)
    width = max(1, max(need))
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    pages = torch.full((len(order), ps * R.TOKEN), 255, dtype=torch.uint8, device=DEV)
    keys = []
    for b, n in enumerate(lens):
        rows = rnd(n, R.ROW, seed=seed * 1000 + b) if fill is None else fill(b, n)
        t = torch.arange(n, device=DEV)
        slots = i32(table[b])[t // ps].long() * ps + t % ps if n else t
        P.paged_cache_write_fp4(rows, slots.int(), pages)
        keys.append(R.held(rows))
    return pages, i32(table), keys


def same(got, want):
    """Equal values, NaN where NaN."""
    got, want = got.double(), want.double()
    off = ~((got == want) | (got.isnan() & want.isnan()))
    at = off.nonzero()[:4].tolist()
    assert not at, [(i, float(got[tuple(i)]), float(want[tuple(i)])) for i in at] + [int(off.sum())]


# --------------------------------------------------------------------------- block format
def test_every_bf16_value_as_a_blocks_largest():
    """Each of the 65,536 bf16 bit patterns as the first value of a block, 31 smaller ones beside it:
    the bytes stand for the nearest values, blocks with inf or NaN read as NaN, reading is exact."""
    bits = torch.arange(65536, device=DEV, dtype=torch.int32)
    g = torch.Generator(device=DEV).manual_seed(3)
    top = bits.to(torch.int16).view(BF).float()
    x = (torch.rand(65536, 32, device=DEV, generator=g) * 2 - 1) * torch.nan_to_num(top, 1.0, 1.0, 1.0)[:, None]
    x = x.to(BF)
    x[:, 0] = bits.to(torch.int16).view(BF)
    # ties: halves of the code steps at the block's own scale
    x[:, 1] = (x[:, 0].float() / 8).to(BF)
    x[:, 2] = (x[:, 0].float() * 0.4375).to(BF)
    rows = torch.cat([x.view(4096, 512), rnd(4096, 64)], 1)
    pages = torch.zeros(64, 64 * R.TOKEN, dtype=torch.uint8, device=DEV)
    slots = torch.randperm(4096, device=DEV).int()
    P.paged_cache_write_fp4(rows, slots, pages)
    want = R.held(rows)
    same(R.stored(pages, slots, 64), want)
    same(P.paged_cache_read_fp4(pages, slots), want)


def test_every_code_between_its_neighbours():
    """Values on a fine grid through one block scale: nearest code, ties to the even one."""
    y = torch.arange(0, 256, device=DEV) / 32 - 3.96875
    rows = torch.zeros(16, R.ROW, device=DEV)
    rows[:, :512] = y.repeat(32).view(16, 512)
    rows[:, 0:512:32] = 6.0
    rows = rows.to(BF)
    pages = torch.zeros(2, 16 * R.TOKEN, dtype=torch.uint8, device=DEV)
    P.paged_cache_write_fp4(rows, torch.arange(16, device=DEV).int(), pages)
    assert torch.equal(P.paged_cache_read_fp4(pages, torch.arange(16, device=DEV).int()).double(), R.held(rows))


@pytest.mark.parametrize("ps", [1, 2, 16, 64, 1024])
@pytest.mark.parametrize("n", [1, 3, 130])
def test_write_and_read_by_slots(ps, n):
    """Rows of a wider matrix into scattered slots of one layer of a page-major pool: the slots' bytes,
    and no others, change; reading them back, unwritten and left-out ones, is exact."""
    n_pages = max(3, 2 * n // ps + 1)
    layers = torch.full((n_pages, 3, ps * R.TOKEN), 9, dtype=torch.uint8, device=DEV)
    pages = layers[:, 1]
    g = torch.Generator(device=DEV).manual_seed(n)
    slots = torch.randperm(n_pages * ps, device=DEV, generator=g)[:n].int()
    rows = rnd(n, 3648, seed=n)[:, 3648 - R.ROW:]
    if n > 2:
        slots[1] = -1
        slots[n - 1] = -7
    P.paged_cache_write_fp4(rows, slots, pages)
    want = torch.full((n_pages * ps, R.ROW), -1.0, dtype=torch.float64, device=DEV)
    live = slots >= 0
    want[slots[live].long()] = R.held(rows)[live]
    untouched = torch.ones(n_pages * ps, dtype=torch.bool, device=DEV)
    untouched[slots[live].long()] = False
    every = torch.arange(n_pages * ps, device=DEV)
    got = R.stored(pages, every, ps)
    assert torch.equal(got[~untouched], want[~untouched])
    nine = R.stored(torch.full((1, R.TOKEN), 9, dtype=torch.uint8, device=DEV), torch.zeros(1, device=DEV), 1)
    assert torch.equal(got[untouched], nine.expand(int(untouched.sum()), -1))
    assert int((layers[:, 0] != 9).sum()) == 0 and int((layers[:, 2] != 9).sum()) == 0
    out = torch.full((n, 600), 5.0, dtype=BF, device=DEV)
    back = P.paged_cache_read_fp4(pages, slots, out=out[:, :R.ROW])
    assert torch.equal(back[live].double(), R.held(rows)[live])
    assert int((back[~live] != 0).sum()) == 0 and int((out[:, R.ROW:] != 5.0).sum()) == 0


def test_the_same_row_written_to_one_slot_many_times():
    """A padded batch repeats its last row and slot."""
    rows, slots = rnd(1, R.ROW).expand(300, R.ROW), i32([37] * 300)
    pages = pool(4, 16, fill=9)
    P.paged_cache_write_fp4(rows, slots, pages)
    same(P.paged_cache_read_fp4(pages, slots), R.held(rows))
    want = torch.full_like(pages, 9)
    P.paged_cache_write_fp4(rows[:1], slots[:1], want)
    assert torch.equal(pages, want)


@pytest.mark.parametrize("n", [8191, 8192, 8193, 8207, 20000])
def test_reads_of_many_rows(n):
    """Rows by the fours and their remainders, slots of no row and past the pool among them, into a wider matrix."""
    ps, n_pages = 32, 700
    pages = pool(n_pages, ps)
    g = torch.Generator(device=DEV).manual_seed(n)
    slots = torch.randint(0, n_pages * ps, (n,), device=DEV, generator=g).int()
    slots[::97] = -1 - slots[::97]
    slots[[0, 5, 4098, n - 2]] = i32([n_pages * ps, 2 ** 31 - 1, n_pages * ps + 7, n_pages * ps])
    out = torch.full((n + 1, 600), 5.0, dtype=BF, device=DEV)
    got = P.paged_cache_read_fp4(pages, slots, out=out[:n, 8:8 + R.ROW])
    live = (slots >= 0) & (slots < n_pages * ps)
    want = torch.where(live[:, None], R.stored(pages, slots.clamp(0, n_pages * ps - 1), ps), 0.0)
    assert torch.equal(got.double(), want)
    assert int((out[:, :8] != 5).sum()) + int((out[:, 8 + R.ROW:] != 5).sum()) + int((out[n] != 5).sum()) == 0
    with pytest.raises(RuntimeError, match="outside the pool"):
        P.check_paged_status()


def test_more_rows_than_a_launch_has_threads_for():
    """2^26 + 1 slots of one row: the first, some around each 2^25 and the last are slots of the pool."""
    n, pages = 2 ** 26 + 1, pool(2, 16, fill=9)
    at = [0, 2 ** 25 - 1, 2 ** 25, 2 ** 25 + 1, 2 ** 26 - 1, 2 ** 26]
    slots = torch.full((n,), -1, dtype=torch.int32, device=DEV)
    slots[at] = i32([3, 0, 31, 16, 7, 20])
    row = rnd(1, R.ROW)
    P.paged_cache_write_fp4(row.expand(n, R.ROW), slots, pages)
    want = pool(2, 16, fill=9)
    P.paged_cache_write_fp4(row.expand(6, R.ROW), slots[at], want)
    assert torch.equal(pages, want)


def test_slots_outside_the_pool_are_skipped_and_reported():
    pages = pool(4, 16, fill=1)
    before = pages.clone()
    P.paged_cache_write_fp4(rnd(3, R.ROW), i32([64, 2 ** 31 - 1, -2 ** 31]), pages)
    assert torch.equal(pages, before)
    with pytest.raises(RuntimeError, match="outside the pool"):
        P.check_paged_status()
    got = P.paged_cache_read_fp4(pages, i32([64, 2 ** 31 - 1, -1]))
    assert int((got != 0).sum()) == 0
    with pytest.raises(RuntimeError, match="outside the pool"):
        P.check_paged_status()


def test_a_pool_past_four_gigabytes():
    """Slots whose byte offsets pass 32 bits: written, read and attended."""
    ps, n_pages = 64, 200_000  # 5.1 GB
    pages = torch.empty(n_pages, ps * R.TOKEN, dtype=torch.uint8, device=DEV)
    n = 100
    table = i32([[n_pages - 1, 3]])
    slots, _, _ = P.paged_slot_map(i32([0]), i32([n]), table, ps, n)
    rows = rnd(n, R.ROW)
    P.paged_cache_write_fp4(rows, slots, pages)
    assert torch.equal(P.paged_cache_read_fp4(pages, slots).double(), R.held(rows))
    q = rnd(1, 16, R.ROW, seed=1, std=0.3)
    got = P.attention_decode_paged_fp4(q, pages, table, i32([n]), SCALE)
    want, tol = R.attention(q[0], R.held(rows), n, SCALE)
    assert ((got[0].double() - want).abs() <= tol).all()


# --------------------------------------------------------------------------- block tables, slot maps
def _state(alloc):
    return i32(alloc.lens + [alloc.head, alloc.count])


@pytest.mark.parametrize("n,ps,width,pages,cap", [(1, 64, 4, 9, 300), (5, 16, 7, 40, 90), (64, 32, 9, 400, 4000),
                                                  (257, 1, 11, 1500, 900), (300, 64, 3, 500, 20000),
                                                  (4096, 16, 4, 9000, 30000), (3, 1024, 2, 5, 3000)])
def test_steps_follow_the_plain_allocator(n, ps, width, pages, cap):
    """Random growth, truncation and retirement for several steps, pages, table columns and slots
    running out at times; each step run twice on the same state."""
    rng = random.Random(n * ps)
    ring = list(range(pages))
    rng.shuffle(ring)
    ref = R.Allocator([0] * n, [[-5] * width for _ in range(n)], ring, rng.randrange(pages), pages, ps)
    table, free, state = i32(ref.table), i32(ring), _state(ref)
    errors = 0
    for k in range(8):
        room = width * ps
        delta = []
        for b in range(n):
            kind = rng.random()
            if kind < 0.35:
                delta.append(1)
            elif kind < 0.6:
                delta.append(rng.randint(0, max(1, min(room, 2 * cap // n))))
            elif kind < 0.75:
                delta.append(-ref.lens[b])
            elif kind < 0.9:
                delta.append(-rng.randint(0, 2 * ps))
            else:
                delta.append(0)
        d = i32(delta)
        first = P.paged_cache_step(state, d, table, free, ps, cap)
        after, slots, positions, rows = P.paged_cache_step(state, d, table, free, ps, cap)
        want, e = ref.step(delta, cap)
        errors |= e
        assert all(torch.equal(x, y) for x, y in zip(first, (after, slots, positions, rows)))
        assert after.tolist() == ref.lens + [ref.head, ref.count], k
        assert [slots.tolist(), positions.tolist(), rows.tolist()] == want, k
        assert free.tolist() == ref.ring and table.tolist() == ref.table, k
        held = [p for b in range(n) for p in ref.table[b][:ref.pages(ref.lens[b])]]
        spare = [ref.ring[(ref.head + i) % pages] for i in range(ref.count)]
        assert sorted(held + spare) == list(range(pages))
        state = after
    if errors:
        with pytest.raises(RuntimeError, match="were skipped"):
            P.check_paged_status()


def test_step_refuses_what_does_not_fit_request_by_request():
    ps, width = 16, 4
    ref = R.Allocator([64, 60, 0, 3, 0, 0], [list(range(4)), list(range(4, 8)), [9] * 4, [8, 9, 9, 9], [9] * 4, [9] * 4],
                      list(range(10, 40)), 7, 3, ps)
    table, free, state = i32(ref.table), i32(ref.ring), _state(ref)
    # past the width; within a page; three pages; within a page; a page too many; a page, but none is left
    delta = [1, 4, 48, 13, 1, 1]
    after, slots, positions, rows = P.paged_cache_step(state, i32(delta), table, free, ps, 100)
    want, _ = ref.step(delta, 100)
    assert [slots.tolist(), positions.tolist(), rows.tolist()] == want and after.tolist()[:6] == [64, 64, 48, 16, 0, 0]
    with pytest.raises(RuntimeError, match="outgrew its block table; no free page"):
        P.check_paged_status()
    huge = [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 0, 2 ** 31 - 1, -1]
    ref2 = R.Allocator(ref.lens, ref.table, ref.ring, ref.head, ref.count, ps)
    after2, slots, positions, rows = P.paged_cache_step(after, i32(huge), table, free, ps, 100)
    want, _ = ref2.step(huge, 100)
    assert after2.tolist() == ref2.lens + [ref2.head, ref2.count] and slots.tolist() == want[0]
    with pytest.raises(RuntimeError, match="outgrew"):
        P.check_paged_status()
    # more tokens than slots: the request that passes them and those after it wait
    after3, slots, _, rows = P.paged_cache_step(after2, i32([0, 5, 0, 0, 9, 1]), table, free, ps, 10)
    assert after3.tolist()[:6] == [64, 5, 48, 16, 0, 0] and rows.tolist() == [1] * 5 + [-1] * 5
    with pytest.raises(RuntimeError, match="max_tokens"):
        P.check_paged_status()


def test_step_and_slot_map_of_the_most_tokens_a_call_may_have():
    """max_tokens of 2^31 - 1, and requests that ask for more together: the later one is refused."""
    most = 2 ** 31 - 1
    table, free = i32([[0, 0], [0, 0], [0, 0]]), i32([2, 1, 0])
    after, slots, _, _ = P.paged_cache_step(i32([0, 0, 0, 0, 3]), i32([3, most, 2]), table, free, 16, most)
    assert after.tolist() == [3, 0, 0, 1, 2] and slots[:3].tolist() == [32, 33, 34] and int(slots[3:].max()) == -1
    with pytest.raises(RuntimeError, match="outgrew its block table; there were more new tokens"):
        P.check_paged_status()
    del slots
    torch.cuda.empty_cache()
    slots, _, rows = P.paged_slot_map(i32([0, 0, 1]), i32([1, most, most]), table, 16, most)
    assert slots[:33].tolist() == [32] + [i % 16 for i in range(32)] and int(slots[33:].max()) == -1
    assert rows[:34].tolist() == [0] + [1] * 32 + [-1]
    with pytest.raises(RuntimeError, match="outside the pool or block table; there were more new tokens"):
        P.check_paged_status()
    del slots, rows
    torch.cuda.empty_cache()


def test_step_reports_every_reason_when_its_sums_are_full():
    """A request that passes the table with the largest delta, one behind it (of the same thread's) past max_tokens."""
    n = 300
    delta = [0] * n
    delta[0], delta[1] = 2 ** 31 - 1, 1
    after, slots, _, _ = P.paged_cache_step(i32([0] * n + [0, 2]), i32(delta), i32([[0]] * n), i32([0, 1]), 16, 50)
    assert after.tolist() == [0] * n + [0, 2] and slots.tolist() == [-1] * 50
    with pytest.raises(RuntimeError, match="outgrew its block table; there were more new tokens"):
        P.check_paged_status()


def test_step_with_corrupt_state_stays_in_bounds():
    """A ring position, a count or a length out of range, a page number that is none: nothing outside
    the tensors is touched, the slots are -1 and the status says so."""
    guard = torch.full((3, 64), -3, dtype=torch.int32, device=DEV)
    table, free = guard[1, :8].view(2, 4), guard[2, :6]
    P.paged_cache_step(i32([-9, 2 ** 31 - 1, -4, 2 ** 31 - 1]), i32([5, -3]), table, free, 16, 8)
    P.paged_cache_step(i32([3, 64, 99, -8]), i32([2, -64]), table, free, 16, 8)
    assert int((guard[0] != -3).sum()) == 0 and int((guard[1, 8:] != -3).sum()) == 0
    assert int((guard[2, 6:] != -3).sum()) == 0
    with pytest.raises(RuntimeError, match="outside the pool"):
        P.check_paged_status()


@pytest.mark.parametrize("n", [1, 7, 256, 4096])
def test_slot_map_of_ranges(n):
    ps, width = 32, 6
    rng = random.Random(n)
    table = [[rng.randrange(1000) for _ in range(width)] for _ in range(n)]
    starts = [rng.randint(0, 60) for _ in range(n)]
    counts = [rng.choice([0, 0, 1, rng.randint(0, 100), -4]) for _ in range(n)]
    want = [(table[b][t // ps] * ps + t % ps, t, b) for b in range(n) for t in range(starts[b], starts[b] + counts[b])]
    total = len(want)
    got = P.paged_slot_map(i32(starts), i32(counts), i32(table), ps, total + 4)
    assert [list(x) for x in zip(*(want + [(-1,) * 3] * 4))] == [x.tolist() for x in got]
    if total > 1:
        short = P.paged_slot_map(i32(starts), i32(counts), i32(table), ps, total - 1)
        assert [x.tolist() for x in short] == [x.tolist()[:total - 1] for x in got]
        with pytest.raises(RuntimeError, match="more new tokens"):
            P.check_paged_status()


def test_slot_map_out_of_range():
    table = i32([[3, -1], [4, 2 ** 30]])
    slots, positions, rows = P.paged_slot_map(i32([-2, 15]), i32([3, 20]), table, 16, 30)
    assert slots.tolist() == [-1] * 3 + [4 * 16 + 15] + [-1] * 26
    with pytest.raises(RuntimeError, match="outside the pool or block table"):
        P.check_paged_status()


# --------------------------------------------------------------------------- attention
def check(q, pages, table, lens, keys, nq=None, scale=SCALE, **kw):
    """Attention of q [T, H, 576] against 64 bits, request by request."""
    cu = None
    if nq is not None:
        cu = i32([sum(nq[:b]) for b in range(len(nq) + 1)])
        kw = {"max_q": max(1, max(nq)), **kw}
    got = P.attention_decode_paged_fp4(q, pages, table, i32(lens), scale, cu, **kw)
    t = 0
    for b, n in enumerate(nq or [1] * len(lens)):
        for j in range(n):
            want, tol = R.attention(q[t], keys[b], lens[b] - n + j + 1, scale)
            off = (got[t].double() - want).abs()
            assert (off <= tol).all(), (b, j, lens[b], float((off / tol.clamp(min=1e-300)).max()))
            t += 1
    return got


@pytest.mark.parametrize("ps", [1, 16, 64, 1024])
@pytest.mark.parametrize("lens", [[1], [0], [31, 32, 33, 0, 64], [63, 65, 127, 128, 129, 1, 5], [700, 0, 2049, 17]])
def test_attention_lengths_and_pages(ps, lens):
    pages, table, keys = batch(lens, ps, seed=len(lens))
    check(rnd(len(lens), 16, R.ROW, seed=5, std=0.3), pages, table, lens, keys)


@pytest.mark.parametrize("heads", [1, 3, 8, 16, 17, 40, 128])
@pytest.mark.parametrize("nq", [[1, 1, 1], [3, 0, 5], [1, 2, 9]])
def test_attention_heads_and_queries(heads, nq):
    """Odd head counts; drafts of several tokens, one request without any, one with more of them than
    it has tokens (the first ones then see nothing)."""
    lens = [200, 70, 6]
    pages, table, keys = batch(lens, 16, seed=heads)
    check(rnd(sum(nq), heads, R.ROW, seed=heads, std=0.3), pages, table, lens, keys, nq)


@pytest.mark.parametrize("lens", [[20000], [9000, 10, 15001], [513] * 40 + [12345], [2048] * 300])
def test_attention_long_and_many(lens):
    pages, table, keys = batch(lens, 64, seed=7)
    check(rnd(len(lens), 16, R.ROW, seed=6, std=0.3), pages, table, lens, keys)


@pytest.mark.parametrize("live", [[0, 1, 4095], [63, 64, 65, 1000, 2047], [4095], list(range(5, 4096, 130))])
def test_attention_of_few_live_rows_among_many_idle_ones(live):
    lens = [0] * 4096
    for i, b in enumerate(live):
        lens[b] = 1 + 37 * i
    pages, table, keys = batch([lens[b] for b in live], 16, seed=len(live))
    wide = torch.full((4096, table.shape[1]), -1, dtype=torch.int32, device=DEV)
    wide[live] = table
    q = rnd(4096, 16, R.ROW, seed=3, std=0.3)
    got = P.attention_decode_paged_fp4(q, pages, wide, i32(lens), SCALE)
    assert int((got[[b for b in range(4096) if not lens[b]]] != 0).sum()) == 0
    for i, b in enumerate(live):
        want, tol = R.attention(q[b], keys[i], lens[b], SCALE)
        assert ((got[b].double() - want).abs() <= tol).all(), b


@pytest.mark.parametrize("requests", [2, 63, 64, 65, 127, 128, 129, 192, 513])
@pytest.mark.parametrize("drafts", [False, True])
def test_attention_numbers_of_requests(requests, drafts):
    """Lengths, empty ones among them, and query counts that differ from request to request."""
    lens = [(b * 29) % 71 if b % 5 else 0 for b in range(requests)]
    lens[-1] = 300
    nq = [(b * 7) % 4 for b in range(requests)] if drafts else None
    pages, table, keys = batch(lens, 32, seed=requests)
    check(rnd(sum(nq) if drafts else requests, 4, R.ROW, seed=requests, std=0.3), pages, table, lens, keys, nq)


def test_attention_of_the_most_requests():
    """65,535 requests of up to 40 tokens, a third of them empty, in pages of one pool that they take by turns."""
    B, ps, n_pages = 65535, 16, 5000
    pages = pool(n_pages, ps)
    keys = R.stored(pages, torch.arange(n_pages * ps, device=DEV), ps)
    g = torch.Generator(device=DEV).manual_seed(4)
    table = torch.randint(0, n_pages, (B, 3), device=DEV, generator=g).int()
    lens = torch.randint(-20, 41, (B,), device=DEV, generator=g).clamp(min=0).int()
    q = rnd(B, 2, R.ROW, seed=5, std=0.3)
    got = P.attention_decode_paged_fp4(q, pages, table, lens, SCALE)
    assert int((got[lens == 0] != 0).sum()) == 0
    t = torch.arange(40, device=DEV)
    for b in list(range(0, B, 211)) + [B - 2, B - 1]:
        n = int(lens[b])
        slots = table[b].long()[t[:n] // ps] * ps + t[:n] % ps
        want, tol = R.attention(q[b], keys[slots], n, SCALE)
        assert ((got[b].double() - want).abs() <= tol).all(), b


def test_attention_of_a_chunk_among_many_requests_with_wide_tables():
    """A prompt's chunk beside decoding rows: 250 requests with room for 163,840 tokens each, 600 queries at most,
    700 of them in all."""
    B, width, ps = 250, 2560, 64
    lens = [(37 * b) % 90 if b % 3 else 0 for b in range(B)]
    nq = [1 if n else 0 for n in lens]
    lens[100], nq[100] = 900, 533
    pages, table, keys = batch(lens, ps, seed=3)
    wide = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    q = rnd(sum(nq), 16, R.ROW, seed=9, std=0.3)
    cu = i32([sum(nq[:b]) for b in range(B + 1)])
    got = P.attention_decode_paged_fp4(q, pages, wide, i32(lens), SCALE, cu, 600)
    t = 0
    for b, n in enumerate(nq):
        for j in range(n):
            if n == 1 or j % 41 == 0 or j == n - 1:
                want, tol = R.attention(q[t], keys[b], lens[b] - n + j + 1, SCALE)
                assert ((got[t].double() - want).abs() <= tol).all(), (b, j)
            t += 1


def _numbered(b, n):
    """Rows whose every 16 tokens have a value in a latent channel of their own (shared by each 512th such tile, the
    values taking turns), and rotary keys that spell the token's number in +-1, each bit three times."""
    t = torch.arange(n, device=DEV)
    x = torch.zeros(n, R.ROW, device=DEV)
    tile = t // 16
    x[t, tile % 512] = torch.tensor(R.VALUES[1:], device=DEV)[(tile // 512 + tile + b) % 7]
    bits = (t[:, None] >> torch.arange(20, device=DEV)) & 1
    x[:, 512:572] = (2.0 * bits - 1).repeat(1, 3)
    return x.to(BF)


CUT = [([4000, 2500, 7003], [9, 3, 5], 8), ([4000, 2500, 7003], [9, 3, 5], 17), ([1999, 8000], [7, 4], 40),
       ([20000], None, 16), ([9000, 10, 15001], None, 16), ([150001], None, 16), ([70003], [3], 16),
       ([300, 6000, 40], [1, 200, 1], 16), ([2048] * 60, None, 16), ([700] * 600, None, 16)]


@pytest.mark.parametrize("lens,nq,heads", CUT)
def test_attention_counts_every_tile_once(lens, nq, heads):
    """All scores equal: an output channel is the sum of its tiles' values over the tokens seen, and one tile more or
    less shows.  Items of one and of many column groups, cut into up to 256 pieces."""
    pages, table, keys = batch(lens, 64, seed=len(lens), fill=_numbered)
    T = sum(nq) if nq else len(lens)
    cu = i32([sum(nq[:b]) for b in range(len(lens) + 1)]) if nq else None
    got = P.attention_decode_paged_fp4(torch.zeros(T, heads, R.ROW, dtype=BF, device=DEV), pages, table, i32(lens),
                                       SCALE, cu, max(nq) if nq else 1)
    t = 0
    for b, n in enumerate(nq or [1] * len(lens)):
        for j in range(n):
            seen = lens[b] - n + j + 1
            want = keys[b][:seen, :512].sum(0) / seen
            # weights of exactly 1, sums of halves below 2^23: the division's rounding and the output's
            off = (got[t].double() - want).abs()
            assert (off <= (2.0 ** -8 + 2.0 ** -20) * want).all(), (b, j, float((off / want.clamp(min=1e-9)).max()))
            t += 1


@pytest.mark.parametrize("lens,nq,heads", CUT)
def test_attention_finds_one_token_each(lens, nq, heads):
    """Every (query token, head) asks for one token, by its number: its output is that token's latent, whichever
    piece, column group and request it is in."""
    rng = random.Random(heads)
    pages, table, keys = batch(lens, 64, seed=len(lens), fill=lambda b, n: torch.cat(
        [rnd(n, 512, seed=b), _numbered(b, n)[:, 512:]], 1))
    at, want = [], []
    for b, n in enumerate(nq or [1] * len(lens)):
        for j in range(n):
            seen = lens[b] - n + j + 1
            pick = [rng.choice([rng.randrange(seen), 16 * rng.randrange(-(-seen // 16)), seen - 1]) for _ in range(heads)]
            at.append(pick)
            want.append(keys[b][pick, :512])
    q = torch.zeros(len(at), heads, R.ROW, device=DEV)
    bits = (torch.tensor(at, device=DEV)[..., None] >> torch.arange(20, device=DEV)) & 1
    # a token of another number scores at least 2 * 3 * 128 * SCALE = 88 less
    q[..., 512:572] = 128 * (2.0 * bits - 1).repeat(1, 1, 3)
    cu = i32([sum(nq[:b]) for b in range(len(lens) + 1)]) if nq else None
    got = P.attention_decode_paged_fp4(q.to(BF), pages, table, i32(lens), SCALE, cu, max(nq) if nq else 1)
    assert torch.equal(got.double(), torch.stack(want))


@pytest.mark.parametrize("std", [0.0, 3.0, 30.0])
def test_attention_flat_and_sharp(std):
    """Equal scores, and scores whose softmax has one token left; a scale of its own."""
    lens = [300, 1100]
    pages, table, keys = batch(lens, 64, seed=2)
    check(rnd(2, 16, R.ROW, seed=3, std=std), pages, table, lens, keys, scale=0.07)


def test_attention_rising_scores():
    """Each tile's scores above all before it: the running maximum moves every time."""
    def fill(b, n):
        x = rnd(n, R.ROW, seed=b)
        x[:, 512:] = torch.linspace(-20, 20 + b, n, device=DEV)[:, None].to(BF)
        return x

    lens = [3000, 257]
    pages, table, keys = batch(lens, 32, fill=fill)
    q = rnd(2, 16, R.ROW, seed=4, std=0.1)
    q[:, :8, 512:] = 0.4
    q[:, 8:, 512:] = -0.4
    check(q, pages, table, lens, keys)


def test_attention_strides():
    """Queries and outputs inside wider tensors, a block table inside a wider one, page-major layers."""
    lens, ps = [40, 333, 90], 32
    pages, table, keys = batch(lens, ps, seed=1)
    layers = torch.full((pages.shape[0], 2, pages.shape[1]), 255, dtype=torch.uint8, device=DEV)
    layers[:, 1] = pages
    wide = torch.full((3, table.shape[1] + 5), 10 ** 9, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    q = rnd(16, 3, 640, seed=9, std=0.3).transpose(0, 1)[:, :, 64:]
    out = torch.full((3, 20, 520), 7.0, dtype=BF, device=DEV)
    got = check(q, layers[:, 1], wide[:, :table.shape[1]], lens, keys, out=out[:, 2:18, :512])
    assert got.data_ptr() == out[:, 2:18].data_ptr()
    assert int((out[:, :2] != 7).sum()) + int((out[:, 18:] != 7).sum()) + int((out[:, :, 512:] != 7).sum()) == 0


@pytest.mark.parametrize("tokens,heads", [(1, 16), (5, 1), (1, 1)])
def test_attention_of_one_token_or_head_takes_any_stride_of_it(tokens, heads):
    lens = [90, 1, 33, 0, 20][:tokens]
    pages, table, keys = batch(lens, 16)
    kept = rnd(tokens, heads, R.ROW, seed=tokens, std=0.3)
    odd = (4 if tokens == 1 else heads * 584, 3 if heads == 1 else 584, 1)
    q = torch.zeros(tokens * heads * 584, dtype=BF, device=DEV).as_strided((tokens, heads, R.ROW), odd)
    q.copy_(kept)
    room = torch.full((tokens * heads * 520,), 7.0, dtype=BF, device=DEV)
    out = room.as_strided((tokens, heads, 512), (4 if tokens == 1 else heads * 520, 3 if heads == 1 else 520, 1))
    got = check(q, pages, table, lens, keys, out=out)
    assert torch.equal(got, P.attention_decode_paged_fp4(kept, pages, table, i32(lens), SCALE))


def test_attention_leaves_query_tokens_of_no_request():
    lens = [50, 60]
    pages, table, keys = batch(lens, 16)
    q = rnd(7, 16, R.ROW, std=0.3)
    out = torch.full((7, 16, 512), 7.0, dtype=BF, device=DEV)
    P.attention_decode_paged_fp4(q, pages, table, i32(lens), SCALE, i32([1, 3, 5]), 2, out)
    assert int((out[0] != 7).sum()) == 0 and int((out[5:] != 7).sum()) == 0
    for t, (b, seen) in enumerate([(0, 49), (0, 50), (1, 59), (1, 60)]):
        want, tol = R.attention(q[1 + t], keys[b], seen, SCALE)
        assert ((out[1 + t].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("what", ["latent", "latent_inf", "rope", "q"])
def test_attention_nan_reaches_only_those_who_see_it(what):
    """A NaN or an infinity in the last cached token: the queries before it stay as they are."""
    lens, nq = [100, 40], [3, 2]

    def fill(b, n):
        x = rnd(n, R.ROW, seed=b)
        if b == 0:
            if what.startswith("latent"):
                x[-1, 100] = float("nan") if what == "latent" else float("-inf")
            elif what == "rope":
                x[-1, 520] = float("nan")
        return x

    pages, table, keys = batch(lens, 32, fill=fill)
    q = rnd(5, 16, R.ROW, std=0.3)
    if what == "q":
        q[2, 4, 7] = float("nan")
    got = P.attention_decode_paged_fp4(q, pages, table, i32(lens), SCALE, i32([0, 3, 5]), 3)
    t = 0
    for b, n in enumerate(nq):
        for j in range(n):
            want, tol = R.attention(q[t], keys[b], lens[b] - n + j + 1, SCALE)
            bad = want.isnan().any(-1)  # a NaN score makes the whole head NaN
            assert torch.equal(bad, torch.tensor([t == 2 and (what != "q" or h == 4) for h in range(16)], device=DEV))
            assert got[t][bad].isnan().all()
            assert ((got[t].double() - want).abs() <= tol)[~bad].all()
            t += 1


@pytest.mark.parametrize("scale,size", [(1e30, 1.0), (0.125, 2.0 ** 33), (0.125, 2.0 ** 70), (1e-30, 2.0 ** 60),
                                        (1e-42, 1.0)])
@pytest.mark.parametrize("n", [1, 200, 5000])
def test_attention_scores_of_any_size(scale, size, n):
    """Scores that pass fp32 when scaled, whose fp32 steps are wider than exp2's range, and hardly any scores at all.
    Each is one product, so exact; the two largest are equal."""
    t = torch.arange(n, device=DEV)
    x = rnd(n, R.ROW, seed=n)
    x[:, 512:] = 0
    x[:, 512] = ((1 + (t % 128) / 128) * torch.exp2((t // 128).float() - 20)).to(BF)
    x[0, 512] = x[-1, 512]
    x = x[torch.randperm(n, device=DEV, generator=torch.Generator(device=DEV).manual_seed(n))]
    pages = torch.zeros(-(-n // 64), 64 * R.TOKEN, dtype=torch.uint8, device=DEV)
    P.paged_cache_write_fp4(x, t.int(), pages)
    q = torch.zeros(1, 16, R.ROW, device=DEV)
    q[0, :, 512] = torch.where(torch.arange(16, device=DEV) % 2 > 0, -size, size)
    q = q.to(BF)
    table = torch.arange(pages.shape[0], device=DEV).int()[None]
    got = P.attention_decode_paged_fp4(q, pages, table, i32([n]), scale)
    keys = R.held(x)
    p = torch.softmax(q[0].double() @ keys.T * scale, -1)
    want, mass = p @ keys[:, :512], p @ keys[:, :512].abs()
    # the output's rounding and the weights' (2^-8 each); differences, scaling, exp2 and fp32 sums 2^-16
    assert ((got[0].double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 * 1.01 + 2.0 ** -16) * mass).all()


def test_attention_weights_add_up_to_one():
    """One token far above the rest, p of which is anything up to 2^8 for the maximum that its wave kept from an
    earlier tile: its rounding must not scale the output.  Two tokens count, 0 with latents 4 and 128 (the same
    wave's next tile) with 6 and a weight 2^5 to 2^8 times as large, so o = 6 - 2w."""
    heads, n = 128, 129
    x = torch.zeros(n, R.ROW, device=DEV)
    x[:, :512] = 6.0
    x[0, :512] = 4.0
    x[1:128, 513] = -2.0 ** 14
    x[128, 512] = 64.0
    pages = torch.zeros(3, 64 * R.TOKEN, dtype=torch.uint8, device=DEV)
    P.paged_cache_write_fp4(x.to(BF), torch.arange(n, device=DEV).int(), pages)
    q = torch.zeros(1, heads, R.ROW, device=DEV)
    q[0, :, 512] = torch.linspace(5, 7.9, heads, device=DEV) * 0.6931471805599453 / 64 / 0.125
    q[0, :, 513] = 1.0
    q = q.to(BF)
    got = P.attention_decode_paged_fp4(q, pages, i32([[0, 1, 2]]), i32([n]), 0.125)
    keys = x.to(BF).double()
    p = torch.softmax(q[0].double() @ keys.T * 0.125, -1)
    want = p @ keys[:, :512]
    # the output's rounding (steps of 2^-5 between 4 and 8, half of one), each weight's to bf16 about the output
    # (2^-8), fp32 sums, exp2 and division (2^-18)
    spread = (p[:, :, None] * (keys[None, :, :512] - want[:, None]).abs()).sum(1)
    tol = 2.0 ** -6 + 2.0 ** -8 * spread + 2.0 ** -18 * 6
    off = (got[0].double() - want).abs()
    assert (off <= tol).all(), float((off / tol).max())


def test_attention_infinite_scores():
    """Scores of -inf count nothing; nothing but them is NaN, and so is a score of +inf."""
    def fill(b, n):
        x = rnd(n, R.ROW, seed=b)
        x[:, 512:] = 0
        at = {0: [3, 40], 1: list(range(n)), 2: [50]}[b]
        x[at, 512] = float("-inf") if b < 2 else float("inf")
        return x

    lens = [60, 33, 64]
    pages, table, keys = batch(lens, 16, fill=fill)
    q = rnd(3, 16, R.ROW, std=0.3)
    q[:, :, 512] = 1.0
    got = P.attention_decode_paged_fp4(q, pages, table, i32(lens), SCALE)
    keep = [t for t in range(60) if t not in (3, 40)]
    want, tol = R.attention(q[0], keys[0][keep], 58, SCALE)
    assert ((got[0].double() - want).abs() <= tol).all()
    assert got[1].isnan().all() and got[2].isnan().all()


def test_attention_skips_bad_pages_and_reports_them():
    """Table entries that name no page hold tokens of zeros; lengths past the table stop at its end."""
    lens = [100, 64]
    pages, table, keys = batch(lens, 32)
    table[0, 1] = pages.shape[0]
    table[0, 3] = -2
    keys[0][32:64] = 0
    keys[0][96:] = 0
    q = rnd(2, 16, R.ROW, std=0.3)
    check(q, pages, table, lens, keys)
    with pytest.raises(RuntimeError, match="outside the pool"):
        P.check_paged_status()
    table[0, 1], table[0, 3] = table[1, 0], table[1, 1]
    keys[0][32:64] = keys[1][:32]
    k0 = torch.cat([keys[0][:96], keys[1][32:64]])
    got = P.attention_decode_paged_fp4(q, pages, table, i32([2 ** 31 - 1, -5]), SCALE)
    want, tol = R.attention(q[0], k0, 128, SCALE)
    assert ((got[0].double() - want).abs() <= tol).all() and int((got[1] != 0).sum()) == 0


def test_attention_more_queries_than_max_q():
    lens = [64]
    pages, table, keys = batch(lens, 32)
    q = rnd(4, 16, R.ROW, std=0.3)
    out = torch.full((4, 16, 512), 7.0, dtype=BF, device=DEV)
    P.attention_decode_paged_fp4(q, pages, table, i32(lens), SCALE, i32([0, 4]), 2, out)
    for t in range(2):
        want, tol = R.attention(q[t], keys[0], 61 + t, SCALE)
        assert ((out[t].double() - want).abs() <= tol).all()
    assert int((out[2:] != 7).sum()) == 0
    with pytest.raises(RuntimeError, match="max_q"):
        P.check_paged_status()


def test_attention_is_the_same_every_time_and_on_every_stream():
    """Same bits for the same call, alone or beside another one on a second stream."""
    lens = [5000, 77, 3001, 900]
    pages, table, _ = batch(lens, 64, seed=4)
    q, q2 = rnd(4, 16, R.ROW, std=0.3), rnd(4, 16, R.ROW, seed=8, std=0.3)
    n = i32(lens)
    first, second = (P.attention_decode_paged_fp4(x, pages, table, n, SCALE) for x in (q, q2))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(side):
            b = P.attention_decode_paged_fp4(q2, pages, table, n, SCALE)
        a = P.attention_decode_paged_fp4(q, pages, table, n, SCALE)
        torch.cuda.synchronize()
        assert torch.equal(a, first) and torch.equal(b, second)


def test_check_sees_calls_on_every_stream():
    """The check waits for work that is still queued on a stream other than the current one."""
    pages = pool(4, 16, fill=1)
    rows, slots = rnd(3, R.ROW), i32([64, 0, 1])
    busy = torch.zeros(1 << 28, device=DEV)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            busy.add_(1)
        P.paged_cache_write_fp4(rows, slots, pages)
    with pytest.raises(RuntimeError, match="outside the pool"):
        P.check_paged_status()
    torch.cuda.synchronize()
    P.check_paged_status()


# --------------------------------------------------------------------------- together
def test_serving_loop_eager_and_captured():
    """Requests join, grow, are rolled back and end while one captured step (lengths, write, attention)
    is replayed between eager calls; every step's output against 64 bits, pages never shared."""
    ps, width, n_pages, rows = 16, 8, 40, 5
    rng = random.Random(1)
    ring = list(range(n_pages))
    rng.shuffle(ring)
    state = i32([0] * rows + [3, n_pages])
    free, table = i32(ring), torch.full((rows, width), -1, dtype=torch.int32, device=DEV)
    pages = torch.full((n_pages, ps * R.TOKEN), 255, dtype=torch.uint8, device=DEV)
    delta, new, q = i32([0] * rows), rnd(rows, R.ROW), rnd(rows, 16, R.ROW, std=0.3)
    keys = [torch.zeros(0, R.ROW, dtype=torch.float64, device=DEV) for _ in range(rows)]

    def step(max_tokens, x):
        after, slots, _, _ = P.paged_cache_step(state, delta, table, free, ps, max_tokens)
        P.paged_cache_write_fp4(x, slots, pages)
        state.copy_(after)
        return P.attention_decode_paged_fp4(q, pages, table, state[:rows], SCALE), slots

    def expect(out, d, x):
        at = 0
        for b in range(rows):
            if d[b] > 0:
                keys[b] = torch.cat([keys[b], R.held(x[at:at + d[b]])])
                at += d[b]
            elif d[b] < 0:
                keys[b] = keys[b][:max(0, len(keys[b]) + d[b])]
            want, tol = R.attention(q[b], keys[b], len(keys[b]), SCALE)
            assert ((out[b].double() - want).abs() <= tol).all(), b
        assert state.tolist()[:rows] == [len(k) for k in keys]
        held = [p for b in range(rows) for p in table[b, :-(-len(keys[b]) // ps)].tolist()]
        assert len(held) == len(set(held)) and len(held) + int(state[rows + 1]) == n_pages

    def eager(d, seed):
        x = rnd(max(1, sum(v for v in d if v > 0)), R.ROW, seed=seed)
        delta.copy_(i32(d))
        out, _ = step(x.shape[0], x)
        expect(out, d, x)

    eager([20, 0, 33, 7, 0], 11)
    delta.fill_(0)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(rows, new)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        captured, slots = step(rows, new)
    for k in range(6):
        for i in range(4):  # the captured step appends one token to each live request
            live = [1 if len(keys[b]) else 0 for b in range(rows)]
            delta.copy_(i32(live))
            q.copy_(rnd(rows, 16, R.ROW, seed=100 * k + i, std=0.3))
            x = rnd(rows, R.ROW, seed=200 * k + i)
            new.copy_(x)
            graph.replay()
            expect(captured, live, x)
        # eager between the replays: a request joins, one is rolled back, one ends
        d = [0] * rows
        d[k % rows] = -len(keys[k % rows]) if len(keys[k % rows]) else 40
        d[(k + 2) % rows] = -3 if len(keys[(k + 2) % rows]) else 18
        eager(d, 300 + k)
    everything, _, _ = P.paged_slot_map(i32([0] * rows), state[:rows].clone(), table, ps, int(state[:rows].sum()))
    assert torch.equal(P.paged_cache_read_fp4(pages, everything).double(), torch.cat(keys))


def test_calls_on_the_librarys_current_device_only_need_the_tensors():
    """A lone page, a lone request, a lone token: the smallest call of each operator."""
    pages = torch.zeros(1, R.TOKEN, dtype=torch.uint8, device=DEV)
    table, free = i32([[-1]]), i32([0])
    state, slots, pos, rows = P.paged_cache_step(i32([0, 0, 1]), i32([1]), table, free, 1, 1)
    assert state.tolist() == [1, 0, 0] and slots.tolist() == pos.tolist() == rows.tolist() == [0]
    x = rnd(1, R.ROW)
    P.paged_cache_write_fp4(x, slots, pages)
    assert torch.equal(P.paged_cache_read_fp4(pages, slots).double(), R.held(x))
    q = rnd(1, 1, R.ROW)
    got = P.attention_decode_paged_fp4(q, pages, table, state[:1], SCALE)
    assert torch.equal(got[0, 0].double(), R.held(x)[0, :512])


def test_empty_calls():
    pages = pool(2, 16, fill=0)
    e = torch.empty(0, dtype=torch.int32, device=DEV)
    table = torch.empty(0, 3, dtype=torch.int32, device=DEV)
    state, slots, _, _ = P.paged_cache_step(i32([1, 2]), e, table, i32([0, 1]), 16, 3)
    assert state.tolist() == [1, 2] and slots.tolist() == [-1] * 3
    assert P.paged_slot_map(e, e, table, 16, 2)[0].tolist() == [-1] * 2
    P.paged_cache_write_fp4(torch.empty(0, R.ROW, dtype=BF, device=DEV), e, pages)
    assert P.paged_cache_read_fp4(pages, e).shape == (0, R.ROW)
    assert P.attention_decode_paged_fp4(torch.empty(0, 16, R.ROW, dtype=BF, device=DEV), pages, table, e,
                                        SCALE).shape == (0, 16, 512)
    out = P.paged_cache_step(i32([5, 0, 2]), i32([0]), i32([[0, 1]]), i32([0, 1]), 16, 0)
    assert out[0].tolist() == [5, 0, 2] and out[1].shape == (0,)


# --------------------------------------------------------------------------- dsv2lite.PagedLatentCache
def test_paged_latent_cache_beside_the_compressed_one():
    """Prompts and decode steps of two layers through PagedLatentCache, the new rows and absorbed queries by
    dsv2_mla_prepare_qlat into a staging buffer, against 64 bits on the rows that the pages hold and against
    dsv2_mla_decode_rows over a bf16 cache of the same rows."""
    from dsv2lite import DSV2Config, PagedLatentCache
    from dsv2lite.rope import cos_sin_tables

    cfg, B, layers = DSV2Config(), 4, 2
    cache = PagedLatentCache(layers, B, max_len=300, n_pages=24, page_size=32)
    cos, sin = cos_sin_tables(cfg, 512, device=DEV)
    kvw, w_ukt = (rnd(512, seed=1, std=0.1) + 1).to(BF), rnd(16, 512, 128, std=0.05, seed=2)
    ptr = lambda t: t.data_ptr()  # noqa: E731

    def prepare(qkva, positions):
        """Cache rows [n, 576] and queries [n, 16, 576]: every row of the staging buffer a sequence of its own."""
        n = qkva.shape[0]
        rows, q = torch.zeros(n, 576, dtype=BF, device=DEV), torch.zeros(n, 16, 576, dtype=BF, device=DEV)
        base = torch.arange(n, device=DEV) - positions
        _hip.call("dsv2_mla_prepare_qlat", ptr(qkva), 3648, n, ptr(positions), ptr(base), ptr(positions + 1), ptr(kvw),
                  1e-6, ptr(cos), ptr(sin), 512, ptr(w_ukt), ptr(rows), ptr(q), None, _hip.stream_ptr())
        return rows, q

    for step, delta in enumerate([[70, 5, 0, 130], [1, 1, 0, 1], [1, 1, 33, 1], [1, -6, 1, 1], [1, 0, 1, 1]]):
        n = sum(d for d in delta if d > 0)
        slots, positions, rows_of = cache.step(i32(delta), n)
        lens = cache.lens.tolist()
        for layer in range(layers):
            new, q = prepare(rnd(n, 3648, seed=10 * step + layer), positions)
            cache.write(layer, new, slots)
            assert torch.equal(cache.read(layer, slots).double(), R.held(new))
            # the last new token of each request that grew asks; the others ask with the first token's query
            last = [max([i for i, b in enumerate(rows_of.tolist()) if b == r], default=0) for r in range(B)]
            qb = q[last]
            got = cache.attend(layer, qb, cfg.softmax_scale)
            every, _, _ = cache.slots_of(torch.zeros_like(cache.lens), cache.lens, sum(lens))
            held = cache.read(layer, every)
            keys = held.double().split(lens)
            base = i32([sum(lens[:b]) for b in range(B)]).long()
            plain = torch.zeros(B, 8192, dtype=BF, device=DEV)
            _hip.call("dsv2_mla_decode_rows", ptr(qb), ptr(held), ptr(base), ptr(cache.lens - 1), ptr(cache.lens), B,
                      cfg.softmax_scale, ptr(plain), 8192, _hip.stream_ptr())
            for b in range(B):
                want, tol = R.attention(qb[b], keys[b], lens[b], cfg.softmax_scale)
                assert ((got[b].double() - want).abs() <= tol).all(), (step, layer, b)
                if lens[b]:
                    assert ((got[b].double() - plain[b].view(16, 512).double()).abs() <= 2 * tol).all(), (step, layer, b)
    assert cache.lens.tolist() == [74, 1, 35, 134] and cache.free_tokens() == (24 - 3 - 1 - 2 - 5) * 32
    cache.check_status()


def test_paged_latent_cache_snapshot_and_overflow():
    from dsv2lite import PagedLatentCache

    cache = PagedLatentCache(1, 3, max_len=64, n_pages=5, page_size=16)
    slots, _, _ = cache.step(i32([20, 30, 1]), 51)
    rows = rnd(51, R.ROW)
    cache.write(0, rows, slots)
    snap = cache.snapshot()
    first = cache.step(i32([-20, 2, 15]), 17)
    assert cache.lens.tolist() == [0, 32, 16] and cache.free_tokens() == 2 * 16
    cache.restore(snap)
    again = cache.step(i32([-20, 2, 15]), 17)
    assert all(torch.equal(x, y) for x, y in zip(first, again))
    assert torch.equal(cache.read(0, slots[20:50]).double(), R.held(rows[20:50]))
    cache.check_status()
    cache.step(i32([33, 0, 49]), 82)  # a page too many; past max_len
    assert cache.lens.tolist() == [0, 32, 16]
    with pytest.raises(RuntimeError, match="outgrew its block table; no free page"):
        cache.check_status()


def test_queries_of_a_step_with_idle_requests_eager_and_captured():
    """The new tokens' queries stand without gaps, whoever is idle, ends or is refused between them: every replay
    of a captured step gives each the attention over its own request."""
    from dsv2lite import PagedLatentCache

    B, most, max_q, ps = 5, 9, 4, 16
    cache = PagedLatentCache(1, B, max_len=96, n_pages=16, page_size=ps)
    slots, _, _ = cache.step(i32([30, 0, 17, 60, 1]), 108)
    first = rnd(108, R.ROW, seed=1)
    cache.write(0, first, slots)
    keys = list(R.held(first).split([30, 0, 17, 60, 1]))
    delta, new, q = i32([0] * B), rnd(most, R.ROW, seed=2), rnd(most, 16, R.ROW, seed=3, std=0.3)
    out = torch.zeros(most, 16, 512, dtype=BF, device=DEV)

    def step():
        slots, _, rows = cache.step(delta, most)
        cache.write(0, new, slots)
        cache.attend(0, q, SCALE, cache.cu_q, max_q, out)
        return rows

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows = step()
    deltas = [[1, 0, 1, 0, 1], [0, 0, 4, 1, 0], [1, 2, -18, 1, 3], [-31, 1, 0, 0, 1], [0, 1, 2, 4, 1], [4, 0, -4, 0, 4],
              [1, 0, 0, 4, 1], [0, 0, 0, 0, 0], [1, 1, 1, 1, 1]]
    for k, d in enumerate(deltas):
        delta.copy_(i32(d))
        new.copy_(rnd(most, R.ROW, seed=10 + k))
        q.copy_(rnd(most, 16, R.ROW, seed=30 + k, std=0.3))
        out.fill_(7.0)
        if k == 3:
            rows_now = step()  # an eager one among the replays
        else:
            graph.replay()
            rows_now = rows
        held, at = R.held(new), 0
        for b in range(B):
            keys[b] = torch.cat([keys[b], held[at:at + d[b]]]) if d[b] > 0 else keys[b][:max(0, len(keys[b]) + d[b])]
            for j in range(max(d[b], 0)):
                assert int(rows_now[at]) == b
                want, tol = R.attention(q[at], keys[b], len(keys[b]) - d[b] + j + 1, SCALE)
                assert ((out[at].double() - want).abs() <= tol).all(), (k, b, j)
                at += 1
        assert int((out[at:] != 7).sum()) == 0 and cache.lens.tolist() == [len(x) for x in keys]
        cache.check_status()
    # one that outgrows its room keeps its places among the others'
    full, others = 96 - len(keys[3]) + 1, [1, 1, 0, 0, 1]
    delta.copy_(i32(others[:3] + [full] + others[4:]))
    big = rnd(full + 3, 16, R.ROW, seed=60, std=0.3)
    x = rnd(full + 3, R.ROW, seed=61)
    slots, _, rows_now = cache.step(delta, full + 3)
    cache.write(0, x, slots)
    got = cache.attend(0, big, SCALE, cache.cu_q, full)
    assert rows_now.tolist() == [0, 1] + [-1] * full + [4]
    for at, b in ((0, 0), (1, 1), (full + 2, 4)):
        keys[b] = torch.cat([keys[b], R.held(x[at:at + 1])])
        want, tol = R.attention(big[at], keys[b], len(keys[b]), SCALE)
        assert ((got[at].double() - want).abs() <= tol).all(), b
    with pytest.raises(RuntimeError, match="outgrew"):
        cache.check_status()


@pytest.mark.parametrize("n", [0, 1, 5, 300, 513, 4096])
def test_step_says_where_each_requests_new_tokens_begin(n):
    """Idle, shrinking, refused and huge requests; the step's other outputs as without it."""
    rng = random.Random(n)
    delta = [rng.choice([0, 1, 1, 3, -2, 40]) for _ in range(n)]
    for later in ([], [2 ** 31 - 1, 5, 2 ** 31 - 1, 0, 7]):
        delta[n - len(later):] = later[:n]
        ends = [0]
        for d in delta:
            ends.append(min(ends[-1] + max(d, 0), 2 ** 31 - 1))
        state, free = i32([1] * n + [0, 9]), i32(list(range(9)) + [-1] * n)
        table = (torch.arange(n, device=DEV) + 9).int()[:, None].repeat(1, 2)
        cu = torch.full((n + 3,), 7, dtype=torch.int32, device=DEV)
        got = P.paged_cache_step(state, i32(delta), table.clone(), free.clone(), 16, 50, cu_q=cu[1:-1])
        plain = P.paged_cache_step(state, i32(delta), table.clone(), free.clone(), 16, 50)
        assert cu.tolist() == [7] + ends + [7] and all(torch.equal(x, y) for x, y in zip(got, plain))
    if n:
        with pytest.raises(RuntimeError, match="outgrew"):
            P.check_paged_status()


def test_a_captured_step_through_the_c_abi_with_padded_rows():
    """Lengths, new rows and queries from projected hidden states, pages and attention as a host would call them, idle
    requests and padding (positions of -1) among the rows; the staging buffer's other rows stay as they are."""
    from dsv2lite import DSV2Config
    from dsv2lite.rope import cos_sin_tables

    cfg, B, most, ps, n_pages, width, max_q = DSV2Config(), 4, 7, 16, 30, 6, 3
    cos, sin = cos_sin_tables(cfg, 128, device=DEV)
    kvw, w_ukt = (rnd(512, seed=1, std=0.1) + 1).to(BF), rnd(16, 512, 128, std=0.05, seed=2)
    pages = torch.full((n_pages, ps * R.TOKEN), 255, dtype=torch.uint8, device=DEV)
    table, ring = torch.full((B, width), -1, dtype=torch.int32, device=DEV), torch.arange(n_pages, device=DEV).int()
    state, after, delta, cu, status = i32([0] * B + [0, n_pages]), i32([0] * (B + 2)), i32([0] * B), i32([0] * (B + 1)), i32([0])
    slots, positions, rows, cap = (i32([0] * most) for _ in range(4))
    base, index = torch.zeros(most, dtype=torch.int64, device=DEV), torch.arange(most, device=DEV)
    qkva, staged = rnd(most, 3648), torch.zeros(most, R.ROW, dtype=BF, device=DEV)
    q, olat = torch.zeros(most, 16, R.ROW, dtype=BF, device=DEV), torch.zeros(most, 16, 512, dtype=BF, device=DEV)
    ws = torch.empty(_hip.lib.dsv2_mla_paged_workspace_size(), dtype=torch.uint8, device=DEV)
    p = lambda t: t.data_ptr()  # noqa: E731

    def step():
        st = _hip.stream_ptr()
        _hip.call("dsv2_paged_step_queries", p(state), p(delta), B, p(table), width, width, p(ring), n_pages, ps, most,
                  p(after), p(slots), p(positions), p(rows), p(cu), p(status), st)
        torch.sub(index, positions, out=base)
        torch.add(positions, 1, out=cap)
        _hip.call("dsv2_mla_prepare_qlat", p(qkva), 3648, most, p(positions), p(base), p(cap), p(kvw), 1e-6, p(cos),
                  p(sin), 128, p(w_ukt), p(staged), p(q), None, st)
        _hip.call("dsv2_paged_write_fp4", p(staged), R.ROW, most, p(slots), p(pages), ps * R.TOKEN, n_pages, ps,
                  p(status), st)
        _hip.call("dsv2_mla_decode_paged_fp4", p(q), 16 * R.ROW, R.ROW, most, 16, p(pages), ps * R.TOKEN, n_pages, ps,
                  p(table), width, width, p(after), B, p(cu), max_q, SCALE, p(olat), 16 * 512, 512, p(ws), ws.numel(),
                  p(status), st)
        state.copy_(after)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    keys = [torch.zeros(0, R.ROW, dtype=torch.float64, device=DEV) for _ in range(B)]
    for k, d in enumerate([[3, 0, 1, 2], [1, 0, 1, 1], [0, 3, -1, 1], [1, 1, 0, 1], [3, 1, 0, -2], [1, 1, 3, 1]] + [[3, 0, 3, 1]] * 5):
        delta.copy_(i32(d))
        qkva.copy_(rnd(most, 3648, seed=70 + k))
        staged.fill_(3.0)
        olat.fill_(7.0)
        if k == 3:
            step()
        else:
            graph.replay()
        new = sum(max(x, 0) for x in d)
        assert positions.tolist()[new:] == [-1] * (most - new) and int((staged[new:] != 3).sum()) == 0
        assert int((staged[:new] != 3).any(1).sum()) == new and int((olat[new:] != 7).sum()) == 0
        held, at = R.held(staged), 0
        for b in range(B):
            keys[b] = torch.cat([keys[b], held[at:at + d[b]]]) if d[b] > 0 else keys[b][:max(0, len(keys[b]) + d[b])]
            for j in range(max(d[b], 0)):
                want, tol = R.attention(q[at], keys[b], len(keys[b]) - d[b] + j + 1, SCALE)
                assert ((olat[at].double() - want).abs() <= tol).all(), (k, b, j)
                at += 1
        assert state.tolist()[:B] == [len(x) for x in keys] and status.tolist() == [0]


def test_a_cache_reports_its_own_errors_only():
    """Two caches of one device: the one that lost tokens says so, whoever is asked first, and the functions' common
    word stays clear."""
    from dsv2lite import PagedLatentCache

    good, full = (PagedLatentCache(1, 2, max_len=64, n_pages=3, page_size=16) for _ in range(2))
    slots, _, _ = good.step(i32([20, 1]), 21)
    full.step(i32([64, 1]), 65)  # a page too many
    good.write(0, rnd(21, R.ROW), slots)
    good.check_status()
    P.check_paged_status()
    with pytest.raises(RuntimeError, match="no free page"):
        full.check_status()
    full.check_status()
    full.read(0, i32([48]))
    good.check_status()
    with pytest.raises(RuntimeError, match="outside the pool"):
        full.check_status()


@pytest.mark.parametrize("name", ["step", "slots", "write", "read", "attention"])
def test_each_function_reports_to_the_word_that_it_is_given(name):
    pages, st = pool(3, 16, fill=0), i32([0])
    {"step": lambda: P.paged_cache_step(i32([16, 0, 3]), i32([1]), i32([[0]]), i32([1, 2, 0]), 16, 1, status=st),
     "slots": lambda: P.paged_slot_map(i32([15]), i32([2]), i32([[0]]), 16, 2, status=st),
     "write": lambda: P.paged_cache_write_fp4(rnd(1, R.ROW), i32([48]), pages, status=st),
     "read": lambda: P.paged_cache_read_fp4(pages, i32([48]), status=st),
     "attention": lambda: P.attention_decode_paged_fp4(rnd(1, 16, R.ROW), pages, i32([[3]]), i32([5]), SCALE,
                                                       status=st)}[name]()
    P.check_paged_status()
    with pytest.raises(RuntimeError, match="outgrew" if name == "step" else "outside the pool"):
        P.check_paged_status(status=st)
    P.check_paged_status(status=st)
    assert st.tolist() == [0]
