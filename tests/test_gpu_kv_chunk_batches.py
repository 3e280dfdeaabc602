"""Attention of chunks where a batch, its values or its weights are uneven."""

from __future__ import annotations

import math

import pytest
import torch

import batched_refs as ref
import paged_refs as pref

pytestmark = pytest.mark.gpu

BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
# how far off the weights over e4m3 pages are: rounded to bf16; of fp16 rows the upper 8 bits, and their rest rounded
E4M3_WEIGHT = {BF16: ref.HALF[BF16], F16: 2.0 ** -7 * ref.HALF[BF16]}


@pytest.fixture(scope="module")
def nat():
    from pocketlm_amd import native

    assert native.native_paged_kv_available(), "libpocketlm_hip.so must load"
    return native


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def attend(nat, q, caches, scales, table, lengths, starts, **kw):
    if caches[0].dtype in (E4M3, torch.uint8):
        return nat.kv_paged_attention_chunk_e4m3(q, *caches, *scales, table.cuda(), i32(lengths), i32(starts), **kw)
    return nat.kv_paged_attention_chunk(q, *caches, table.cuda(), i32(lengths), i32(starts), **kw)


def randn(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("at", [0, 7, 15])
def test_sequences_without_rows_change_nothing(nat, e4m3, at):
    """A prompt beside sequences with a long history and no rows in the call is cut as it is alone: the same bits."""
    heads, kvh, dim, page, rows = 28, 4, 128, 16, 500
    caches, scales, table = pref.make_pages([rows], page, kvh, dim, E4M3 if e4m3 else BF16, 1)
    q = randn((rows, heads, dim), BF16, 2)
    want = attend(nat, q, caches, scales, table, [0], [0, rows])
    wide = torch.full((16, 20000 // page), -7, dtype=torch.int32)
    wide[at, :table.shape[1]] = table[0]
    lengths = [0 if b == at else 20000 - b for b in range(16)]
    got = attend(nat, q, caches, scales, wide, lengths, [0] * (at + 1) + [rows] * (16 - at))
    assert torch.equal(got, want)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("length,rows", [(150, 20), (0, 170), (100, 1)])
def test_values_at_the_end_of_bf16(nat, e4m3, length, rows):
    """Averages of values of 2^125 stay finite where scores rise by a little after the first positions.

    Position 100 has a score of 5 (2^7.2 times the others' weight), so the weights, as shares of the largest, sum to
    at most 1 + 170 / 147: times 1.75 * 2^125 below 2^128."""
    heads, kvh, dim, page = 4, 2, 64, 16
    caches, scales, table = pref.make_pages([length + rows], page, kvh, dim, E4M3 if e4m3 else BF16, 3)
    k, v = (c.view(torch.uint8) if e4m3 else c for c in caches)
    k.zero_()
    five = torch.tensor(5.0).to(E4M3).view(torch.uint8).cuda() if e4m3 else 5.0
    if length + rows > 100:
        k[int(table[0, 100 // page]), 100 % page, :, 0] = five
    if e4m3:
        v.copy_((256.0 + 192.0 * torch.rand(v.shape, generator=torch.Generator().manual_seed(4))).to(E4M3).view(torch.uint8))
        scales[0].fill_(1.0)
        scales[1].fill_(2.0 ** 117)
    else:
        v.copy_(((1.0 + 0.75 * torch.rand(v.shape, generator=torch.Generator().manual_seed(4))) * 2.0 ** 125).to(BF16))
    q = torch.zeros((rows, heads, dim), dtype=BF16, device="cuda")
    q[:, :, 0] = 1.0
    got = attend(nat, q, caches, scales, table, [length], [0, rows], softmax_scale=1.0)
    want, bound = pref.chunk(q, *caches, table, [length], [0, rows], 1.0, scales=scales)
    assert bool(want.isfinite().all())
    pref.agree(got, want, bound)


def milliseconds(call, times=5):
    """The shortest of a few calls."""
    call()
    best = math.inf
    for _ in range(times):
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        call()
        end.record()
        end.synchronize()
        best = min(best, begin.elapsed_time(end))
    return best


@pytest.mark.parametrize("dtype,e4m3", [(BF16, False), (F16, False), (BF16, True), (F16, True)])
@pytest.mark.parametrize("heads,kvh,dim", [(14, 2, 128), (8, 8, 64), (4, 2, 256)])
@pytest.mark.parametrize("what", ["value", "key", "query", "hidden"])
def test_a_nan_that_rows_see(nat, dtype, e4m3, heads, kvh, dim, what):
    """A prompt whose first position holds a NaN (or an infinity in fp16 values), one NaN query row, and a NaN of the last
    position: the right rows get it, and the call takes no more than a few times as long as without."""
    rows, page = 1400, 16
    caches, scales, table = pref.make_pages([rows], page, kvh, dim, E4M3 if e4m3 else dtype, 5)
    q = randn((rows, heads, dim), dtype, 6)

    def call():
        return attend(nat, q, caches, scales, table, [0], [0, rows])

    usual = milliseconds(call)
    first, last = (int(table[0, 0]), 0), (int(table[0, (rows - 1) // page]), (rows - 1) % page)
    if what == "query":
        q[700, 1, 3] = float("nan")
    else:
        cache = caches[0] if what == "key" else caches[1]
        value = float("inf") if dtype == F16 and what == "value" else float("nan")
        if e4m3:
            cache.view(torch.uint8)[(*(last if what == "hidden" else first), slice(None), 5)] = 0x7F
        else:
            cache[(*(last if what == "hidden" else first), slice(None), 5)] = value
    poisoned = milliseconds(call)
    got = call()
    want, bound = pref.chunk(q, *caches, table, [0], [0, rows], dim ** -0.5, scales=scales,
                             weight=E4M3_WEIGHT[dtype] if e4m3 else None)
    pref.agree(got, want, bound)
    assert poisoned < 10 * usual + 0.2, (poisoned, usual)


@pytest.mark.parametrize("dtype,e4m3", [(BF16, False), (F16, False), (BF16, True), (F16, True)])
@pytest.mark.parametrize("heads,kvh,dim", [(14, 2, 128), (4, 4, 64), (2, 1, 248), (2, 1, 176)])
@pytest.mark.parametrize("length,rows", [(0, 90), (3000, 70), (130, 1200)])
def test_infinities_of_both_signs(nat, dtype, e4m3, heads, kvh, dim, length, rows):
    """One that every row sees, then two of the other sign in the same and in another head value, then a NaN, that later
    rows see; pages that are not there between them, for which rows that hold such values may be read."""
    page = 16
    if e4m3:
        dim -= dim % 16
    caches, scales, table = pref.make_pages([length + rows], page, kvh, dim, E4M3 if e4m3 else dtype, 9, dirt=float("nan"))

    def put(pos, at, value):
        where = (int(table[0, pos // page]), pos % page)
        if not e4m3:
            caches[1][(*where, slice(None), at)] = value
            return
        # a scale of infinity, whose sign is its byte's (and NaN where that is 0): head values of the other sign take one too
        raw = caches[1].view(torch.uint8)
        if math.isnan(value):
            raw[(*where, slice(None), at)] = 0x7F
            return
        raw[where] = 0x38 if value > 0 else 0xB8
        scales[1][where[0], :, where[1]] = math.inf

    put(0, 5, math.inf)
    put(length + rows // 3, 7, -math.inf)
    put(length + rows // 2, 5, -math.inf)
    put(length + rows - 2, dim - 1, math.nan)
    for pos in (32, length + rows // 4):
        if pos // page not in (0, (length + rows // 3) // page):
            table[0, pos // page] = -7
    q = randn((rows, heads, dim), dtype, 10)
    got = attend(nat, q, caches, scales, table, [length], [0, rows])
    want, bound = pref.chunk(q, *caches, table, [length], [0, rows], dim ** -0.5, scales=scales,
                             weight=E4M3_WEIGHT[dtype] if e4m3 else None)
    pref.agree(got, want, bound)
    assert bool(want[0, :, 5].isinf().all()) and bool(want[-1, :, dim - 1].isnan().all())
    if int(table[0, (length + rows // 2) // page]) >= 0:
        assert bool(want[-1, :, 5].isnan().all())


@pytest.mark.parametrize("heads,kvh,dim", [(28, 4, 128), (4, 2, 64), (3, 1, 256), (2, 2, 192)])
@pytest.mark.parametrize("length,rows,place", [(5000, 3, 0), (5000, 3, 2900), (5000, 40, 4999), (1500, 1500, 700), (20000, 130, 12345)])
def test_weight_on_one_of_many_e4m3_positions(nat, heads, kvh, dim, length, rows, place):
    """A row whose weight lies on one position gets that position's value, rounded once: the weight's own rounding does
    not show, however many positions there are.

    The position's score is 24 above the others' bound of 3, so theirs are shares of exp(-21) each, 21500 of them
    2^-15.9 in all; rounded to bf16, 2^-8 of that, of the largest value.  Its own weight has 15 bits."""
    page = 64
    caches, scales, table = pref.make_pages([length + rows], page, kvh, dim, E4M3, 7)
    k = caches[0].view(torch.uint8)
    g = torch.Generator().manual_seed(8)
    # scores: head value 0 of every key at most 3 in size (the others 0), of the chosen one 24
    k.zero_()
    low = (torch.rand(k.shape[:3], generator=g) * 6 - 3).to(E4M3)
    k[..., 0] = low.view(torch.uint8).cuda()
    k[int(table[0, place // page]), place % page, :, 0] = torch.tensor(24.0).to(E4M3).view(torch.uint8).cuda()
    scales[0].fill_(1.0)
    q = torch.zeros((rows, heads, dim), dtype=BF16, device="cuda")
    q[:, :, 0] = (1.0 + 0.25 * torch.rand((rows, heads), generator=g)).to(BF16).cuda()
    got = attend(nat, q, caches, scales, table, [length], [0, rows], softmax_scale=1.0)
    want, bound = pref.chunk(q, *caches, table, [length], [0, rows], 1.0, scales=scales, weight=2.0 ** -15)
    rest = 2.0 ** -8 * (length + rows) * math.exp(-21.0) * 448.0 * float(scales[1].max())
    # the output's own rounding: half a step at its size, not the most that is of any size
    half = torch.exp2(torch.floor(torch.log2(want.abs() * (1 + 2.0 ** -9) + rest)) - 8)
    pref.agree(got, want, bound + rest - ref.HALF[BF16] * want.abs() + half)


@pytest.mark.parametrize("heads,kvh,dim", [(28, 4, 128), (4, 2, 64), (3, 1, 256)])
@pytest.mark.parametrize("length,rows", [(6000, 40), (2500, 500)])
def test_weight_on_a_few_of_many_e4m3_positions(nat, heads, kvh, dim, length, rows):
    """Rows of which two positions, far apart, have a half of the weight each, and their values cancel but for a part.

    Both are in tiles of weights of two values: 15 bits of each, beside 2^-8 of the others, 2 * 6040 exp(-21) at most."""
    page = 32
    caches, scales, table = pref.make_pages([length + rows], page, kvh, dim, E4M3, 11)
    k, v = (c.view(torch.uint8) for c in caches)
    g = torch.Generator().manual_seed(12)
    k.zero_()
    k[..., 0] = (torch.rand(k.shape[:3], generator=g) * 6 - 3).to(E4M3).view(torch.uint8).cuda()
    pair = [(int(table[0, p // page]), p % page) for p in (length // 3, length - 5)]
    for where in pair:
        k[where[0], where[1], :, 0] = torch.tensor(24.0).to(E4M3).view(torch.uint8).cuda()
    v[pair[1]] = v[pair[0]] ^ 0x80  # times its own scale, of up to 9 / 4 of the other
    scales[0].fill_(1.0)
    q = torch.zeros((rows, heads, dim), dtype=BF16, device="cuda")
    q[:, :, 0] = (1.0 + 0.25 * torch.rand((rows, heads), generator=g)).to(BF16).cuda()
    got = attend(nat, q, caches, scales, table, [length], [0, rows], softmax_scale=1.0)
    want, bound = pref.chunk(q, *caches, table, [length], [0, rows], 1.0, scales=scales, weight=2.0 ** -15)
    rest = 2.0 ** -8 * 2 * (length + rows) * math.exp(-21.0) * 448.0 * float(scales[1].max())
    pref.agree(got, want, bound + rest)


def many(sequences, long, page, heads, kvh, dim, dtype, e4m3, seed):
    """(q, caches, scales, table, lengths, starts): short sequences of 0 to 3 rows, idle ones among them, and a few long
    ones, over random pages of a small pool."""
    pool = 200
    caches, scales, _ = pref.make_pages([pool * page], page, kvh, dim, E4M3 if e4m3 else dtype, seed, spare=0)
    g = torch.Generator().manual_seed(seed + 1)
    lengths = [(7 * b) % 150 if b % 11 else -1 for b in range(sequences)]
    rows = [(3 * b) % 4 for b in range(sequences)]
    for at, (length, n) in long.items():
        lengths[at], rows[at] = length, n
    cols = (max(x + r for x, r in zip(lengths, rows)) + page - 1) // page
    table = torch.randint(0, pool, (sequences, cols), generator=g, dtype=torch.int32)
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    return randn((starts[-1] + 3, heads, dim), dtype, seed + 2), caches, scales, table, lengths, starts


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("heads,kvh,dim", [(14, 2, 128), (4, 1, 64), (3, 1, 80)])
@pytest.mark.parametrize("sequences", [62, 63, 256, 257, 300, 1100])
def test_long_sequences_among_many(nat, e4m3, heads, kvh, dim, sequences):
    long = {sequences // 3: (20000, 1), sequences - 1: (9000, 2), 0: (5000, 70)}
    q, caches, scales, table, lengths, starts = many(sequences, long, 16, heads, kvh, dim, BF16, e4m3, sequences)
    got = attend(nat, q, caches, scales, table, lengths, starts)
    want, bound = pref.chunk(q, *caches, table, lengths, starts, dim ** -0.5, scales=scales,
                             weight=E4M3_WEIGHT[BF16] if e4m3 else None)
    pref.agree(got, want, bound)


@pytest.mark.parametrize("sequences", [4000, 8191, 65535])
def test_long_sequences_among_thousands(nat, sequences):
    """Rows of a few sequences against those alone."""
    long = {5: (30000, 1), sequences - 2: (12000, 3)}
    q, caches, scales, table, lengths, starts = many(sequences, long, 16, 4, 1, 64, BF16, False, 3)
    got = attend(nat, q, caches, scales, table, lengths, starts)
    for b in (2, 5, 1001, sequences // 2, sequences - 2, sequences - 1):
        mine = slice(starts[b], starts[b + 1])
        want, bound = pref.chunk(q[mine], *caches, table[b:b + 1], lengths[b:b + 1], [0, starts[b + 1] - starts[b]], 64 ** -0.5)
        pref.agree(got[mine], want, bound)
    assert not bool(got[starts[-1]:].any())


def test_scratch_of_many_sequences(nat):
    """A caller's scratch is not left, whatever the call's sequences are split into."""
    from pocketlm_amd import _lib

    lib = _lib.load()
    heads, kvh, dim, page = 14, 2, 128, 16
    q, caches, scales, table, lengths, starts = many(700, {20: (30000, 1), 600: (4000, 90)}, page, heads, kvh, dim, BF16, False, 8)
    table_d, rows = table.cuda(), q.shape[0]
    need = lib.kv_paged_attention_chunk_scratch_bytes(700, rows, heads, kvh, dim, table.shape[1] * page)
    held = torch.full((need + 65536,), 0xA5, dtype=torch.uint8, device="cuda")
    for ls in (lengths, [x // 50 for x in lengths], [min(x * 30, 20000) for x in lengths], lengths):
        want = attend(nat, q, caches, scales, table, ls, starts)
        out = torch.full_like(q, 7.0)
        lengths_d, starts_d = i32(ls), i32(starts)
        lib.pocketlm_set_stream(torch.cuda.current_stream().cuda_stream)
        assert 0 == lib.kv_paged_attention_chunk_u16(
            q.data_ptr(), caches[0].data_ptr(), caches[1].data_ptr(), table_d.data_ptr(), lengths_d.data_ptr(),
            starts_d.data_ptr(), out.data_ptr(), held.data_ptr(), need, rows, 700, heads, kvh, dim, heads * dim, dim,
            table.shape[1], caches[0].shape[0], page, *caches[0].stride()[:3], dim ** -0.5, 1)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert bool((held[need:] == 0xA5).all())


def test_time_of_one_long_sequence_among_many(nat):
    """It is split over the device as among few: within twice the time (16 times where it is not split)."""
    times = []
    for sequences in (250, 300):
        q, caches, scales, table, lengths, starts = many(sequences, {100: (60000, 1)}, 16, 28, 4, 128, BF16, False, 4)
        where = (table.cuda(), i32(lengths), i32(starts))
        times.append(milliseconds(lambda: nat.kv_paged_attention_chunk(q, *caches, *where)))
    assert times[1] < 2 * times[0], times


def test_many_sequences_in_a_graph(nat):
    """Captured with short lengths, replayed with others that are split, in other orders; rows of no sequence are zero."""
    q, caches, scales, table, lengths, starts = many(400, {7: (30000, 1), 300: (5000, 80)}, 16, 14, 2, 128, BF16, False, 6)
    table_d, lengths_d, starts_d = table.cuda(), i32([50 if x >= 0 else -1 for x in lengths]), i32(starts)

    def call():
        return nat.kv_paged_attention_chunk(q, *caches, table_d, lengths_d, starts_d)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for ls, ss in ((lengths, starts), (lengths[::-1], starts), ([x // 100 for x in lengths], starts), (lengths, [0] * 300 + starts[300:]),
                   (lengths, starts)):
        lengths_d.copy_(i32(ls))
        starts_d.copy_(i32(ss))
        want = call()
        torch.cuda.synchronize()
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("heads,kvh,dim,rows", [(28, 4, 128, 1), (28, 4, 128, 36), (28, 4, 128, 37), (5, 5, 64, 3), (3, 1, 256, 50)])
def test_scratch_of_few_rows(nat, heads, kvh, dim, rows):
    """It holds partials of the columns that the rows have, and no more is written."""
    from pocketlm_amd import _lib

    lib = _lib.load()
    page, length = 16, 30000
    caches, _, table = pref.make_pages([200 * page], page, kvh, dim, BF16, 3, spare=0)
    table = torch.randint(0, 200, (1, (length + rows + page - 1) // page), generator=torch.Generator().manual_seed(1),
                          dtype=torch.int32)
    q = randn((rows, heads, dim), BF16, 4)
    need = lib.kv_paged_attention_chunk_scratch_bytes(1, rows, heads, kvh, dim, table.shape[1] * page)
    # two partials of at most a tile's columns of each of at most 256 runs of all heads, and their plan
    most = min(256 if dim <= 128 else 128, rows * heads // kvh)
    assert 0 < need <= 2 * 256 * most * (dim + 2) * 4 + 65536
    held = torch.full((need + 65536,), 0xA5, dtype=torch.uint8, device="cuda")
    table_d, lengths, starts, out = table.cuda(), i32([length]), i32([0, rows]), torch.zeros_like(q)
    want, bound = pref.chunk(q, *caches, table, [length], [0, rows], dim ** -0.5)
    lib.pocketlm_set_stream(torch.cuda.current_stream().cuda_stream)
    assert 0 == lib.kv_paged_attention_chunk_u16(
        q.data_ptr(), caches[0].data_ptr(), caches[1].data_ptr(), table_d.data_ptr(), lengths.data_ptr(), starts.data_ptr(),
        out.data_ptr(), held.data_ptr(), need, rows, 1, heads, kvh, dim, heads * dim, dim, table.shape[1], caches[0].shape[0], page,
        *caches[0].stride()[:3], dim ** -0.5, 1)
    torch.cuda.synchronize()
    pref.agree(out, want, bound)
    assert bool((held[need:] == 0xA5).all())


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("heads,kvh,dim", [(28, 4, 128), (6, 6, 64), (4, 2, 256), (3, 1, 80)])
@pytest.mark.parametrize("rows,longest", [(3, 2500), (45, 700)])
def test_values_that_are_not_finite_in_some_sequences(nat, e4m3, heads, kvh, dim, rows, longest):
    """Workgroups that go from sequences with such values, seen by all, by some and by few of the rows, to others without
    them, and pages that are not there."""
    page, count = 16, 40
    lengths = [(longest * (7 * b % count)) // count for b in range(count)]
    g = torch.Generator().manual_seed(13)
    starts = list(range(0, rows * count + 1, rows))
    q = torch.randn((rows * count, heads, dim), generator=g).to(BF16).cuda()
    caches, scales, table = pref.make_pages([x + rows for x in lengths], page, kvh, dim, E4M3 if e4m3 else BF16, 14,
                                            dirt=float("nan"))
    v = caches[1].view(torch.uint8) if e4m3 else caches[1]
    bad = 0x7F if e4m3 else float("nan")
    for b in range(0, count, 3):
        for pos, at in ((lengths[b] + rows - 1, 5), (lengths[b] + rows // 2, 7), (lengths[b] // 2, 9)):
            v[int(table[b, pos // page]), pos % page, b % kvh, at] = bad
        if not e4m3:
            v[int(table[b, lengths[b] // page]), lengths[b] % page, :, 11] = float("inf")
    for b in range(0, count, 7):
        if lengths[b] > 200:
            table[b, 3] = -7
    got = attend(nat, q, caches, scales, table, lengths, starts)
    want, bound = pref.chunk(q, *caches, table, lengths, starts, dim ** -0.5, scales=scales,
                             weight=E4M3_WEIGHT[BF16] if e4m3 else None)
    assert bool(want.isnan().any()) and bool(want.isfinite().all(2).any())
    pref.agree(got, want, bound)
