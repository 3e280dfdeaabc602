"""Attention of chunks of new rows over 16-bit and e4m3 pages, and of decode
steps over e4m3 pages, against the definition in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

import batched_refs as ref
import paged_refs as pref

pytestmark = pytest.mark.gpu

BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
# how far off the weights over e4m3 pages are: rounded to bf16; of fp16 rows the upper 8 bits, which leave less than 2^-7,
# and that rest rounded to bf16
E4M3_WEIGHT = {BF16: ref.HALF[BF16], F16: 2.0 ** -7 * ref.HALF[BF16]}


@pytest.fixture(scope="module")
def nat():
    from pocketlm_amd import native

    assert native.native_paged_kv_available(), "libpocketlm_hip.so must load on the GPU box"
    return native


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def starts_of(rows, first=0):
    starts = [first]
    for r in rows:
        starts.append(starts[-1] + r)
    return starts


def attend(nat, q, caches, scales, table, lengths, starts, **kw):
    if caches[0].dtype in (E4M3, torch.uint8):
        return nat.kv_paged_attention_chunk_e4m3(q, *caches, *scales, table.cuda(), i32(lengths), i32(starts), **kw)
    return nat.kv_paged_attention_chunk(q, *caches, table.cuda(), i32(lengths), i32(starts), **kw)


def check(nat, lengths, rows, page, heads, kvh, dim, dtype, *, e4m3=False, seed=0, scale=None, before=0, behind=0, spoil=None,
          make=None, dirt=float("nan"), size=1.0):
    """One call with rows before the first sequence and behind the last one, and `dirt` in every slot that holds none."""
    lens = [max(0, x) + r if x >= 0 else 0 for x, r in zip(lengths, rows)]
    caches, scales, table = pref.make_pages(lens, page, kvh, dim, E4M3 if e4m3 else dtype, seed, dirt=dirt)
    if spoil is not None:
        spoil(table)
    starts = starts_of(rows, before)
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn((starts[-1] + behind, heads, dim), generator=g) * size).to(dtype).cuda()
    if make is not None:
        make(q, caches, scales, table, starts)
    kw = {} if scale is None else {"softmax_scale": scale}
    got = attend(nat, q, caches, scales, table, lengths, starts, **kw)
    want, bound = pref.chunk(q, *caches, table, lengths, starts, dim ** -0.5 if scale is None else scale, scales=scales,
                             weight=E4M3_WEIGHT[dtype] if e4m3 else None)
    assert got.shape == q.shape and got.dtype == dtype
    pref.agree(got, want, bound)
    return got


HEADS = [(28, 4, 128), (4, 2, 64), (7, 1, 128), (6, 3, 96), (3, 3, 80), (8, 1, 256), (2, 2, 192), (5, 5, 16)]


@pytest.mark.parametrize("dtype,e4m3", [(BF16, False), (F16, False), (BF16, True), (F16, True)])
@pytest.mark.parametrize("heads,kvh,dim", HEADS)
def test_heads_and_lengths(nat, dtype, e4m3, heads, kvh, dim):
    """Prompts, chunks and single tokens in one call, sequences without rows, idle ones and rows of none."""
    check(nat, [0, 37, -1, 200, 0, 63, 64], [70, 1, 5, 0, 1, 130, 2], 16, heads, kvh, dim, dtype, e4m3=e4m3, before=3, behind=2)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kvh,dim", [(4, 2, 40), (2, 1, 8), (3, 1, 72), (2, 2, 136), (6, 2, 248)])
def test_16_bit_head_dims(nat, dtype, heads, kvh, dim):
    check(nat, [0, 37, 150], [70, 1, 33], 16, heads, kvh, dim, dtype)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("page", [1, 3, 16, 63, 64, 65, 100, 4096])
def test_page_sizes(nat, e4m3, page):
    check(nat, [0, 5, 300], [65, 64, 3], page, 4, 2, 64, BF16, e4m3=e4m3)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("rows", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257])
def test_rows_at_tiles_borders(nat, e4m3, rows):
    check(nat, [0, 64 - rows % 64, 1], [rows, rows, 1], 16, 2, 2, 128, F16, e4m3=e4m3)


@pytest.mark.parametrize("dtype,e4m3", [(BF16, False), (F16, False), (BF16, True)])
@pytest.mark.parametrize("heads,kvh,dim", [(28, 4, 128), (16, 16, 64), (8, 4, 256), (4, 1, 128)])
def test_few_rows_of_long_sequences(nat, dtype, e4m3, heads, kvh, dim):
    """Positions split over workgroups, in pieces of different numbers for each sequence."""
    check(nat, [5000, 700, 0, 2111], [3, 40, 9, 1], 64, heads, kvh, dim, dtype, e4m3=e4m3, behind=1)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kvh,dim", [(12, 2, 128), (16, 16, 64), (3, 1, 256), (4, 2, 96), (2, 1, 192)])
@pytest.mark.parametrize("lengths,rows", [([0], [2]), ([0, 0], [3, 40]), ([40, 0], [2, 300]), ([500], [9])])
def test_few_positions_over_e4m3_pages(nat, dtype, heads, kvh, dim, lengths, rows):
    """Where a weight may be the whole result its rounding must not show: bounds as of a weight rounded to 15 bits."""
    lens = [x + r for x, r in zip(lengths, rows)]
    caches, scales, table = pref.make_pages(lens, 16, kvh, dim, E4M3, dim)
    starts = starts_of(rows)
    q = (torch.randn((starts[-1], heads, dim), generator=torch.Generator().manual_seed(dim)) * 2).to(dtype).cuda()
    got = attend(nat, q, caches, scales, table, lengths, starts)
    want, bound = pref.chunk(q, *caches, table, lengths, starts, dim ** -0.5, scales=scales, weight=2.0 ** -15)
    pref.agree(got, want, bound)


def test_one_row_of_a_very_long_sequence(nat):
    check(nat, [100000], [1], 256, 4, 2, 64, BF16)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("heads,kvh,dim,rows", [(28, 4, 128, 2500), (64, 8, 64, 1100)])
def test_many_rows(nat, e4m3, heads, kvh, dim, rows):
    """Enough rows for waves of two blocks of columns."""
    check(nat, [0, 321], [rows, rows // 7], 64, heads, kvh, dim, BF16, e4m3=e4m3)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lengths,rows", [([0], [500]), ([0], [1500]), ([0, 0, 0], [900, 3, 860]), ([700], [37]), ([300] * 16, [150] * 16),
                                          ([0, 3800], [300, 2])])
def test_calls_that_whole_tiles_or_runs_take(nat, e4m3, lengths, rows):
    """Sizes on both sides of what decides between whole tiles and runs, with tables that reach further."""
    check(nat, lengths, rows, 16, 14, 2, 128, BF16, e4m3=e4m3, seed=sum(rows))
    check(nat, [*lengths, 5000], [*rows, 1], 16, 14, 2, 128, BF16, e4m3=e4m3, seed=sum(rows))


def test_many_rows_fp16(nat):
    check(nat, [77, 0], [2500, 300], 16, 32, 8, 128, F16)


@pytest.mark.parametrize("sequences", [250, 256, 257, 300, 5000])
def test_many_sequences(nat, sequences):
    rows = [(3 * b) % 4 for b in range(sequences)]
    lengths = [(7 * b) % 90 if b % 11 else -1 for b in range(sequences)]
    check(nat, lengths, rows, 32, 2, 1, 64, BF16, before=2, behind=5)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("long", [False, True])
def test_pages_that_are_not_there(nat, e4m3, long):
    """Entries outside the cache within, at both ends of and all over what a row sees."""
    def spoil(table):
        table[0, 1] = -1
        table[0, 5:9] = 10 ** 6
        table[1, :] = -3
        table[2, 0] = -1
        if long:
            table[3, 100:140] = -2

    check(nat, [100, 30, 0, 3000 if long else 20], [60, 40, 20, 12], 16, 4, 2, 64, BF16, e4m3=e4m3, spoil=spoil)


@pytest.mark.parametrize("e4m3", [False, True])
def test_positions_past_the_table(nat, e4m3):
    """Rows whose sequence is longer than its table see what the table holds."""
    dim, page = 64, 16
    caches, scales, table = pref.make_pages([64, 64], page, 2, dim, E4M3 if e4m3 else BF16, 3, extra_cols=0)
    q = torch.randn((100, 4, dim), generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    lengths, starts = [30, 60], [0, 60, 100]
    got = attend(nat, q, caches, scales, table, lengths, starts)
    want, bound = pref.chunk(q, *caches, table, lengths, starts, dim ** -0.5, scales=scales)
    pref.agree(got, want, bound)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("value", [float("inf"), float("nan"), float("-inf")])
@pytest.mark.parametrize("lengths,rows", [([0, 10], [100, 20]), ([3000], [40]), ([70, 0], [2400, 5])])
def test_infinities_that_only_later_rows_see(nat, dtype, value, lengths, rows):
    """Values and keys of a new row reach that row and the later ones, and no other."""
    heads, kvh = (28, 4) if rows[0] > 1000 else (4, 2)

    def make(q, caches, scales, table, starts):
        for cache, b, back in ((caches[1], 0, rows[0] // 2), (caches[0], 0, 3), (caches[1], 0, 1)):
            pos = lengths[b] + rows[b] - back
            cache[int(table[b, pos // 16]), pos % 16, :, 5] = value

    got = check(nat, lengths, rows, 16, heads, kvh, 64, dtype, make=make)
    assert bool(torch.isfinite(got[:rows[0] // 2]).all())
    assert not bool(torch.isfinite(got[rows[0] - 1]).all())


@pytest.mark.parametrize("lengths,rows", [([0, 10], [100, 20]), ([3000], [40]), ([70, 0], [2400, 5])])
def test_e4m3_nan_that_only_later_rows_see(nat, lengths, rows):
    heads, kvh = (28, 4) if rows[0] > 1000 else (4, 2)

    def make(q, caches, scales, table, starts):
        pos = lengths[0] + rows[0] // 2
        caches[1].view(torch.uint8)[int(table[0, pos // 16]), pos % 16] = 0x7F
        pos = lengths[0] + rows[0] - 2
        scales[0][int(table[0, pos // 16]), :, pos % 16] = float("nan")
        scales[1][int(table[0, pos // 16]), :, pos % 16] = float("inf")

    got = check(nat, lengths, rows, 16, heads, kvh, 64, BF16, e4m3=True, make=make)
    assert bool(torch.isfinite(got[:rows[0] // 2]).all())
    assert not bool(torch.isfinite(got[rows[0] - 1]).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_queries_of_infinities(nat, dtype):
    def make(q, caches, scales, table, starts):
        q[3, 1, 2] = float("inf")
        q[50, 0, 60] = float("nan")

    check(nat, [0, 3], [70, 40], 16, 4, 2, 64, dtype, make=make)


@pytest.mark.parametrize("dtype,e4m3", [(BF16, False), (F16, False), (BF16, True)])
@pytest.mark.parametrize("scale", [-0.125, 0.0, 1.0, 3e-5])
def test_softmax_scales(nat, dtype, e4m3, scale):
    check(nat, [0, 100], [70, 9], 16, 4, 2, 64, dtype, e4m3=e4m3, scale=scale)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_growing_scores(nat, dtype):
    """Scores that rise along the positions move the running maximum in every tile; falling ones leave weights
    that vanish."""
    dim = 64

    def rising(sign):
        def make(q, caches, scales, table, starts):
            q.zero_()
            q[:, :, 0] = 1.0
            caches[0].zero_()
            for b in range(2):
                for pos in range(550):
                    if int(table[b, pos // 16]) >= 0:
                        caches[0][int(table[b, pos // 16]), pos % 16, :, 0] = sign * 4.0 * (pos // 8)
        return make

    for sign in (1.0, -1.0):
        check(nat, [500, 0], [50, 130], 16, 2, 2, dim, dtype, scale=1.0, make=rising(sign))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scores_of_the_type_s_lowest_value_and_minus_infinity(nat, dtype):
    """Scores of -inf give a weight of 0; rows of which every score is -inf are 0 / 0."""
    def make(q, caches, scales, table, starts):
        q.zero_()
        q[:, :, 0] = 1.0
        k = caches[0]
        k[..., 0] = 0.0
        k[int(table[0, 0]), :8, :, 0] = -math.inf       # the first 8 positions of sequence 0
        k[int(table[1, 0]), :4, :, 0] = torch.finfo(dtype).min
        k[..., 1:] = 0.0

    got = check(nat, [0, 0], [40, 40], 16, 2, 2, 64, dtype, make=make)
    assert bool(got[:8].isnan().all()) and bool(torch.isfinite(got[8:]).all())


def test_weights_of_large_scores_in_fp16(nat):
    """Scores past 2^24 have no room for a factor of the weights."""
    def make(q, caches, scales, table, starts):
        q.zero_()
        q[:, :, 0] = 6e4
        caches[0].zero_()
        caches[0][..., 0] = 6e4

    check(nat, [0, 60], [40, 40], 16, 2, 2, 64, F16, scale=1.0, make=make)


@pytest.mark.parametrize("e4m3", [False, True])
def test_other_orders_and_strides(nat, e4m3):
    """[page][head][slot] caches, queries as columns of a projection, scales with strides of their own: the same bits."""
    kvh, heads, dim, page = 2, 6, 64, 8
    lens, starts = [90, 33], [0, 40, 60]
    caches, scales, table = pref.make_pages(lens, page, kvh, dim, E4M3 if e4m3 else BF16, 1)
    lengths = [50, 13]
    qkv = torch.randn((60, (heads + 2 * kvh) * dim), generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
    q = qkv[:, :heads * dim].unflatten(1, (-1, dim))
    first = attend(nat, q.contiguous(), caches, scales, table, lengths, starts)
    raw = [(c.view(torch.uint8) if e4m3 else c).permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for c in caches]
    wide = scales
    if e4m3:
        wide = [torch.full((s.shape[0], 2, kvh, page + 3), 5.0, device="cuda")[:, 1, :, :page] for s in scales]
        for t, s in zip(wide, scales):
            t.copy_(s)
    odd = torch.empty((60, heads, dim + 3), dtype=BF16, device="cuda")[..., 2:dim + 2]
    odd.copy_(q)
    for other in (q, odd):
        assert torch.equal(first, attend(nat, other, raw, wide, table, lengths, starts))


def test_offsets_past_32_bits(nat):
    """Pages beyond 4 GiB of a cache, of 16-bit and of e4m3 values."""
    for e4m3 in (False, True):
        kvh, dim, page = 2, 128, 64
        stride = (1 << 28) + 16  # values of a page
        pages = 20
        shape, strides = (pages, page, kvh, dim), (stride, kvh * dim, dim, 1)
        dtype = torch.uint8 if e4m3 else BF16
        big = [torch.empty(((pages - 1) * stride + page * kvh * dim,), dtype=dtype, device="cuda") for _ in range(2)]
        caches = [t.as_strided(shape, strides) for t in big]
        small, scales, _ = pref.make_pages([pages * page], page, kvh, dim, E4M3 if e4m3 else BF16, 5, spare=0)
        for c, s in zip(caches, small):
            c.copy_(s.view(torch.uint8) if e4m3 else s)
        table = torch.tensor([[19, 0, 17, 18, 1]], dtype=torch.int32)
        g = torch.Generator().manual_seed(6)
        q = torch.randn((30, 4, dim), generator=g).to(BF16).cuda()
        got = attend(nat, q, caches, scales, table, [280], [0, 30])
        want, bound = pref.chunk(q, *(c.view(E4M3) if e4m3 else c for c in small), table, [280], [0, 30], dim ** -0.5,
                                 scales=scales, weight=ref.HALF[BF16])
        pref.agree(got, want, bound)
        if e4m3:
            got = nat.kv_paged_attention_decode_e4m3(q[:1], *caches, *scales, table.cuda(), i32([280]))
            pref.agree(got, want[:1], bound[:1])
            k = torch.randn((2, kvh, dim), generator=g).to(BF16).cuda()
            nat.kv_paged_append_e4m3(None, k, k, *caches, *scales, table.cuda(), i32([18 + 64 * 2]))
            held, _ = pref.gathered(caches[1], scales[1], table[0], 148)
            u, scale, off, _ = pref.quantized(k.double(), torch.zeros_like(k, dtype=torch.float64))
            pref.agree(held[146:148] / scale[..., None], u, off + 1e-6 * u.abs())
        del big, caches


# ---------------------------------------------------------------- decode over e4m3 pages

def check_decode(nat, lengths, rows, page, heads, kvh, dim, dtype, *, seed=0, spoil=None, make=None, dirt=float("nan"),
                 extra=1):
    lens = [x + rows if x >= 0 else 0 for x in lengths]
    caches, scales, table = pref.make_pages(lens, page, kvh, dim, E4M3, seed, dirt=dirt, extra_cols=extra)
    if spoil is not None:
        spoil(table)
    n = len(lengths)
    q = torch.randn((n, rows, heads, dim), generator=torch.Generator().manual_seed(seed + 1)).to(dtype).cuda()
    if make is not None:
        make(q, caches, scales, table)
    got = nat.kv_paged_attention_decode_e4m3(q[:, 0] if rows == 1 else q, *caches, *scales, table.cuda(), i32(lengths))
    # weights in two bf16 halves: 15 bits of each
    want, bound = pref.chunk(q.flatten(0, 1), *caches, table, lengths, [rows * b for b in range(n + 1)], dim ** -0.5,
                             scales=scales, weight=2.0 ** -15)
    pref.agree(got.reshape(want.shape), want, bound)
    return got


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kvh,dim", HEADS + [(4, 2, 48), (2, 1, 112), (3, 1, 240), (16, 8, 64)])
@pytest.mark.parametrize("room", [1, 400])
def test_decode_heads_and_lengths(nat, dtype, heads, kvh, dim, room):
    check_decode(nat, [0, 37, -1, 700, 127, 128, 31], 1, 16, heads, kvh, dim, dtype, extra=room)


@pytest.mark.parametrize("rows", [2, 3, 4, 8])
@pytest.mark.parametrize("heads,kvh,dim", [(28, 4, 128), (8, 8, 64), (4, 1, 256), (14, 2, 64)])
@pytest.mark.parametrize("longest", [300, 9000])
def test_decode_of_several_rows(nat, rows, heads, kvh, dim, longest):
    check_decode(nat, [longest, 5, 0, -3, longest // 2], rows, 32, heads, kvh, dim, BF16)


@pytest.mark.parametrize("page", [1, 7, 100, 1024])
def test_decode_page_sizes(nat, page):
    check_decode(nat, [0, 3000, 99], 2, page, 4, 2, 128, F16)


def test_decode_splits_and_many_sequences(nat):
    check_decode(nat, [40000], 1, 64, 28, 4, 128, BF16)
    check_decode(nat, [(37 * b) % 400 - 3 for b in range(300)], 1, 16, 8, 2, 64, BF16)


def test_decode_pages_that_are_not_there(nat):
    def spoil(table):
        table[0, 1:3] = -1
        table[1, :] = 10 ** 6
        table[2, 60:] = -1

    check_decode(nat, [100, 30, 2000], 3, 16, 4, 2, 64, BF16, spoil=spoil)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_decode_nan_that_only_later_rows_see(nat, dim):
    def make(q, caches, scales, table):
        for b, pos in ((0, 1002), (1, 2)):
            caches[1].view(torch.uint8)[int(table[b, pos // 16]), pos % 16] = 0xFF
            scales[1][int(table[b, (pos + 1) // 16]), :, (pos + 1) % 16] = float("inf")
            scales[0][int(table[b, (pos + 1) // 16]), :, (pos + 1) % 16] = float("nan")

    got = check_decode(nat, [1000, 0], 4, 16, 4, 2, dim, BF16, make=make)
    assert bool(torch.isfinite(got[:, :2]).all()) and bool(got[:, 2:].isnan().any())


def test_decode_scales_of_all_sizes(nat):
    """Scales from 2^-120 to 2^100 in one sequence: weights times scales leave fp16 and stay in fp32."""
    def make(q, caches, scales, table):
        for s in (scales[1],):
            s.copy_(torch.exp2(torch.randint(-120, 100, s.shape, generator=torch.Generator().manual_seed(1)).float()).cuda())
        scales[1][int(table[0, 3]), :, 2] = 2.0 ** 3

    for dtype in (BF16,):
        check_decode(nat, [500], 1, 16, 4, 2, 64, dtype, make=make, dirt=None)


def test_decode_equals_a_chunk_of_single_rows(nat):
    """The two paths over the same pages agree within both bounds."""
    lengths = [700, 5, 0, 130]
    caches, scales, table = pref.make_pages([x + 1 for x in lengths], 16, 4, 128, E4M3, 9)
    q = torch.randn((4, 28, 128), generator=torch.Generator().manual_seed(4)).to(BF16).cuda()
    one = nat.kv_paged_attention_decode_e4m3(q, *caches, *scales, table.cuda(), i32(lengths))
    two = attend(nat, q, caches, scales, table, lengths, list(range(5)))
    _, bound = pref.chunk(q, *caches, table, lengths, list(range(5)), 128 ** -0.5, scales=scales, weight=ref.HALF[BF16])
    pref.agree(one, two.double(), 2 * bound)


# ---------------------------------------------------------------- as they are used

@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prompts_in_chunks_then_tokens(nat, dtype, e4m3):
    """Two conversations: their prompts in uneven chunks, then a few tokens, each step an append with norms and an
    attention; every result against the definition over what the caches hold, and the caches against one append of all."""
    heads, kvh, dim, page = 8, 2, 128, 16
    total = [150, 61]
    steps = [([64, 20], [0, 0]), ([70, 1], [64, 20]), ([1, 38], [134, 21]), ([1, 1], [135, 59]), ([1, -1], [136, 60]),
             ([1, 1], [137, 60])]
    g = torch.Generator().manual_seed(11)
    rows_of = [torch.randn((n, (heads + 2 * kvh) * dim), generator=g).to(dtype).cuda() for n in total]
    wq, wk = ((1 + 0.1 * torch.randn(dim, generator=g)).to(dtype).cuda() for _ in range(2))
    freq = nat.kv_rope_frequencies(dim, 1e6)
    kind = E4M3 if e4m3 else dtype
    caches, scales, table = pref.make_pages(total, page, kvh, dim, kind, 2)
    again, scales2, _ = pref.make_pages(total, page, kvh, dim, kind, 2)
    table_d = table.cuda()

    def append(qkv, caches, scales, lengths, starts):
        q, k, v = (t.unflatten(1, (-1, dim)) for t in qkv.split([heads * dim, kvh * dim, kvh * dim], 1))
        if e4m3:
            return nat.kv_paged_append_e4m3(q, k, v, *caches, *scales, table_d, lengths, q_norm_weight=wq, k_norm_weight=wk,
                                            rms_eps=1e-6, row_starts=starts, rope_frequencies=freq)
        return nat.kv_paged_norm_append(q, k, v, wq, wk, *caches, table_d, lengths, rms_eps=1e-6, row_starts=starts,
                                        rope_frequencies=freq)

    done = [0, 0]
    for rows, lengths in steps:
        lengths = [x if r >= 0 else -1 for x, r in zip(lengths, rows)]
        rows = [max(0, r) for r in rows]
        starts = starts_of(rows)
        qkv = torch.cat([rows_of[b][done[b]:done[b] + rows[b]] for b in range(2)])
        q = append(qkv, caches, scales, i32(lengths), i32(starts))
        got = attend(nat, q, caches, scales, table, lengths, starts)
        want, bound = pref.chunk(q, *caches, table, lengths, starts, dim ** -0.5, scales=scales,
                                 weight=E4M3_WEIGHT[dtype] if e4m3 else None)
        pref.agree(got, want, bound)
        if rows == [1, 1]:
            if e4m3:
                token = nat.kv_paged_attention_decode_e4m3(q, *caches, *scales, table_d, i32(lengths))
            else:
                token = nat.kv_paged_attention_decode(q, *caches, table_d, i32(lengths))
            pref.agree(token, want, bound)
        done = [d + r for d, r in zip(done, rows)]
    append(torch.cat([r[:d] for r, d in zip(rows_of, done)]), again, scales2, i32([0, 0]), i32([0, done[0], sum(done)]))
    for b in range(2):
        for c, d, s, t in zip(caches, again, scales, scales2):
            x, _ = pref.gathered(c, s, table[b], done[b])
            y, _ = pref.gathered(d, t, table[b], done[b])
            assert torch.equal(x, y)


@pytest.mark.parametrize("e4m3", [False, True])
def test_captured_steps_follow_what_is_on_the_device(nat, e4m3):
    """An append and its attention captured once; replays with other rows, lengths and row starts, idle sequences
    among them, equal the eager calls, with eager work between; a second graph over the same caches has its own scratch."""
    heads, kvh, dim, page, rows = 8, 2, 128, 16, 48
    room = [1500, 900, 400]
    kind = E4M3 if e4m3 else BF16
    caches, scales, table = pref.make_pages(room, page, kvh, dim, kind, 5)
    table_d = table.cuda()
    freq = nat.kv_rope_frequencies(dim, 1e4)
    g = torch.Generator().manual_seed(1)
    w = (1 + 0.1 * torch.randn(dim, generator=g)).to(BF16).cuda()
    qkv = torch.zeros((rows, (heads + 2 * kvh) * dim), dtype=BF16, device="cuda")
    lengths, starts = i32([0, 0, 0]), i32([0, 16, 32, 48])

    def step():
        q, k, v = (t.unflatten(1, (-1, dim)) for t in qkv.split([heads * dim, kvh * dim, kvh * dim], 1))
        if e4m3:
            q = nat.kv_paged_append_e4m3(q, k, v, *caches, *scales, table_d, lengths, q_norm_weight=w, k_norm_weight=w,
                                         rms_eps=1e-6, row_starts=starts, rope_frequencies=freq)
            return nat.kv_paged_attention_chunk_e4m3(q, *caches, *scales, table_d, lengths, starts)
        q = nat.kv_paged_norm_append(q, k, v, w, w, *caches, table_d, lengths, rms_eps=1e-6, row_starts=starts,
                                     rope_frequencies=freq)
        return nat.kv_paged_attention_chunk(q, *caches, table_d, lengths, starts)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for turn, (ls, ss) in enumerate([([0, 0, 0], [0, 16, 32, 48]), ([1400, 3, 100], [0, 1, 40, 48]), ([700, -1, 0], [0, 30, 31, 40]),
                                     ([1452, 852, 352], [0, 48, 48, 48]), ([5, 800, 399], [2, 2, 47, 48])]):
        qkv.copy_(torch.randn(qkv.shape, generator=g).to(BF16))
        lengths.copy_(i32(ls))
        starts.copy_(i32(ss))
        want = step()
        torch.cuda.synchronize()
        for graph, out in graphs if turn % 2 else graphs[::-1]:
            out.fill_(7.0)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), turn


def test_calls_on_another_stream(nat):
    heads, kvh, dim = 8, 2, 128
    caches, scales, table = pref.make_pages([900, 300], 16, kvh, dim, E4M3, 7)
    q = torch.randn((60, heads, dim), generator=torch.Generator().manual_seed(3)).to(BF16).cuda()
    lengths, starts = [860, 280], [0, 40, 60]
    want = attend(nat, q, caches, scales, table, lengths, starts)
    one = nat.kv_paged_attention_decode_e4m3(q[:2], *caches, *scales, table.cuda(), i32([860, 280]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append((attend(nat, q, caches, scales, table, lengths, starts),
                        nat.kv_paged_attention_decode_e4m3(q[:2], *caches, *scales, table.cuda(), i32([860, 280]))))
    for s in streams:
        s.synchronize()
    for a, b in got:
        assert torch.equal(a, want) and torch.equal(b, one)


def test_scratch_of_the_caller_and_of_the_library(nat):
    """The C entry takes NULL for its own scratch, and stays within a caller's."""
    from pocketlm_amd import _lib

    lib = _lib.load()
    heads, kvh, dim, page = 28, 4, 128, 16
    caches, _, table = pref.make_pages([5000, 700], page, kvh, dim, BF16, 3)
    table_d, lengths, starts = table.cuda(), i32([4990, 600]), i32([0, 10, 110])
    q = torch.randn((110, heads, dim), generator=torch.Generator().manual_seed(3)).to(BF16).cuda()
    want = nat.kv_paged_attention_chunk(q, *caches, table_d, lengths, starts)
    need = lib.kv_paged_attention_chunk_scratch_bytes(2, 110, heads, kvh, dim, table.shape[1] * page)
    assert need > 0
    held = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device="cuda")

    def call(scratch, nbytes):
        out = torch.zeros_like(q)
        lib.pocketlm_set_stream(torch.cuda.current_stream().cuda_stream)
        code = lib.kv_paged_attention_chunk_u16(q.data_ptr(), caches[0].data_ptr(), caches[1].data_ptr(), table_d.data_ptr(),
                                                lengths.data_ptr(), starts.data_ptr(), out.data_ptr(), scratch, nbytes, 110, 2,
                                                heads, kvh, dim, heads * dim, dim, table.shape[1], caches[0].shape[0], page,
                                                *caches[0].stride()[:3], dim ** -0.5, 1)
        assert code == 0
        torch.cuda.synchronize()
        return out

    assert torch.equal(call(None, 0), want)
    assert torch.equal(call(held.data_ptr(), need), want)
    assert bool((held[need:] == 0xA5).all())


def test_empty_calls(nat):
    caches, scales, table = pref.make_pages([4], 4, 1, 64, E4M3, 0)
    q = torch.empty((0, 1, 64), dtype=F16, device="cuda")
    assert attend(nat, q, caches, scales, table, [0], [0, 0]).shape == (0, 1, 64)
    q = torch.ones((3, 1, 64), dtype=F16, device="cuda")
    got = nat.kv_paged_attention_chunk_e4m3(q, *caches, *scales, table.cuda()[:0], i32([]), i32([0]))
    assert torch.equal(got, torch.zeros_like(q))


def test_row_starts_that_do_not_ascend(nat):
    """No promise about their rows, but the call ends and the next one is right."""
    heads, kvh, dim = 14, 2, 128
    caches, _, table = pref.make_pages([3000, 700, 40], 16, kvh, dim, BF16, 3)
    table_d = table.cuda()
    q = torch.randn((60, heads, dim), generator=torch.Generator().manual_seed(3)).to(BF16).cuda()
    want = nat.kv_paged_attention_chunk(q, *caches, table_d, i32([2970, 680, 30]), i32([0, 30, 50, 60]))
    for starts in ([0, 50, 20, 60], [60, 0, 60, 0], [-5, 1000, -7, 30]):
        got = nat.kv_paged_attention_chunk(q, *caches, table_d, i32([2970, 680, 30]), i32(starts))
        torch.cuda.synchronize()
        assert got.shape == q.shape
    again = nat.kv_paged_attention_chunk(q, *caches, table_d, i32([2970, 680, 30]), i32([0, 30, 50, 60]))
    assert torch.equal(again, want)
