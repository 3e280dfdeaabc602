"""The paged key-value cache: rows appended with their rotation, and the
attention of new rows over the pages, against the definitions in 64 bits; then
the operators of a batched decode step one after another, eagerly and captured."""

from __future__ import annotations

import math

import pytest
import torch

import batched_refs as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nat():
    from pocketlm_amd import native

    assert native.native_paged_kv_available(), "libpocketlm_hip.so must load on the GPU box"
    return native


def i32(values, device="cuda"):
    return torch.tensor(values, dtype=torch.int32, device=device)


# ---------------------------------------------------------------- append

def check_append(nat, lengths, rows, page, heads, kvh, dim, dtype, *, pairs=None, interleaved=False, starts=None,
                 theta=1e4, seed=0, spoil=None):
    """Appends to caches that hold values everywhere and compares every slot."""
    total = sum(rows) if starts is None else starts[-1]
    behind = 3 if starts is not None else 0  # rows behind the last sequence
    g = torch.Generator().manual_seed(seed)
    k_cache, v_cache, table = ref.make_pages([max(0, x) + r for x, r in zip(lengths, rows)], page, kvh, dim, dtype, seed)
    if spoil is not None:
        spoil(table)
    qkv = torch.randn((total + behind, (heads + 2 * kvh) * dim), generator=g).to(dtype)
    q, k, v = (t.unflatten(1, (-1, dim)) for t in qkv.split([heads * dim, kvh * dim, kvh * dim], 1))
    pairs = dim // 2 if pairs is None else pairs
    freq = torch.tensor([theta ** (-2.0 * i / max(1, 2 * pairs)) for i in range(pairs)], dtype=torch.float64)
    dk, dv = k_cache.cuda(), v_cache.cuda()
    rejected = i32([5])
    gq, gk, gv = (t.unflatten(1, (-1, dim)) for t in qkv.cuda().split([heads * dim, kvh * dim, kvh * dim], 1))
    got = nat.kv_paged_append(gq, gk, gv, dk, dv, table.cuda(), i32(lengths),
                              row_starts=None if starts is None else i32(starts),
                              rope_frequencies=freq.cuda() if pairs else None, interleaved=interleaved, rejected=rejected)
    want_q = torch.zeros(q.shape, dtype=torch.float64)
    want_k, bound_q, bound_k = k_cache.double(), torch.zeros(q.shape, dtype=torch.float64), torch.zeros_like(k_cache).double()
    want_v, refused = v_cache.clone(), 0
    for r, where in enumerate(ref.places(table, lengths, total + behind, starts)):
        if where is None:
            continue
        b, pos = where
        yq, eq = ref.rotate(q[r], pos, freq, interleaved)
        want_q[r], bound_q[r] = yq, eq + (ref.HALF[dtype] * (yq.abs() + eq) + ref.TINY[dtype] if pairs else 0)
        index = pos // page
        pid = int(table[b, index]) if index < table.shape[1] else -1
        if not 0 <= pid < k_cache.shape[0]:
            refused += 1
            continue
        yk, ek = ref.rotate(k[r], pos, freq, interleaved)
        want_k[pid, pos % page] = yk
        bound_k[pid, pos % page] = ek + (ref.HALF[dtype] * (yk.abs() + ek) + ref.TINY[dtype] if pairs else 0)
        want_v[pid, pos % page] = v[r]
    ref.within(got, want_q, bound_q, "queries")
    ref.within(dk, want_k, bound_k, "keys")
    assert torch.equal(dv.cpu(), want_v)
    assert int(rejected) == 5 + refused
    return refused


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kvh,dim,pairs,interleaved", [
    (28, 4, 128, None, False), (4, 4, 64, None, True), (6, 1, 256, None, False), (3, 3, 8, None, False),
    (5, 5, 96, None, True), (4, 2, 40, None, False), (4, 2, 72, None, True), (8, 2, 128, 32, False),
    (8, 2, 64, 7, True), (8, 2, 64, 5, False), (4, 4, 80, 0, False), (4, 4, 24, 0, False)])
def test_append_one_to_eight_rows(nat, dtype, heads, kvh, dim, pairs, interleaved):
    for rows in (1, 3, 8):
        lengths = [0, 17, -1, 5, 100003]
        check_append(nat, lengths, [rows] * 5, 7 if dim == 8 else 4096, heads, kvh, dim, dtype, pairs=pairs,
                     interleaved=interleaved, seed=rows) if kvh * dim <= 64 else \
            check_append(nat, lengths[:4] + [403], [rows] * 5, 16, heads, kvh, dim, dtype, pairs=pairs,
                         interleaved=interleaved, seed=rows)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page", [1, 5, 64])
def test_append_prompts_of_ragged_lengths(nat, dtype, page):
    """Sequences without rows, idle ones, and rows behind the last sequence."""
    rows = [40, 0, 1, 77, 9, 0]
    lengths = [0, 3, 31, 0, -2, 8]
    starts = [sum(rows[:i]) for i in range(7)]
    check_append(nat, lengths, rows, page, 4, 2, 64, dtype, starts=starts, seed=page)


def test_append_many_sequences(nat):
    rows = [(3 * b) % 5 for b in range(150)]
    starts = [sum(rows[:i]) for i in range(151)]
    check_append(nat, [b % 37 for b in range(150)], rows, 8, 2, 1, 32, torch.bfloat16, starts=starts)


def test_append_far_positions(nat):
    """Angles of positions beyond 2^24: the caches are one page of a table's far end."""
    dim, far = 64, 2 ** 30 + 12345
    page = 2 ** 20
    table = torch.zeros((1, 2 ** 10 + 1), dtype=torch.int32)
    k_cache = torch.zeros((1, 1, 1, dim), dtype=torch.float16, device="cuda").expand(1, page, 1, dim)
    freq = nat.kv_rope_frequencies(dim, 1e6)
    x = torch.randn((1, 2, dim), generator=torch.Generator().manual_seed(2)).half()
    want, bound = ref.rotate(x[0], far, freq.cpu(), False)
    got = nat.kv_paged_append(x.cuda(), x[:, :1].cuda(), x[:, :1].cuda(), k_cache, k_cache, table.cuda(), i32([far]),
                              rope_frequencies=freq)
    ref.within(got[0], want, bound + ref.HALF[torch.float16] * (want.abs() + bound) + ref.TINY[torch.float16])


def test_append_leaves_rows_without_a_page(nat):
    def spoil(table):
        table[0, 1] = -1
        table[1, 0] = 999

    assert check_append(nat, [6, 2, 9], [8, 8, 8], 4, 2, 2, 16, torch.float16, spoil=spoil) > 0
    # positions past the table
    k = torch.randn((4, 1, 16), dtype=torch.float16, device="cuda")
    cache = torch.zeros((2, 4, 1, 16), dtype=torch.float16, device="cuda")
    v_cache, count = torch.zeros_like(cache), i32([0])
    assert nat.kv_paged_append(None, k, k, cache, v_cache, i32([[1, 0]]), i32([6]), rejected=count) is None
    assert int(count) == 2 and torch.equal(v_cache[0, 2:], k[:2]) and not v_cache[1].any() and not v_cache[0, :2].any()


def test_append_into_other_orders(nat):
    """Caches [page][head][slot], one cache of keys and values, rows at odd addresses."""
    kvh, dim, page, n = 3, 32, 8, 6
    both = torch.zeros((5, 2, kvh, page, dim), dtype=torch.bfloat16, device="cuda")
    k_cache, v_cache = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    raw = torch.randn((n * kvh * dim + 1,), device="cuda").bfloat16()
    k = raw[1:].view(n, kvh, dim)
    v = torch.randn((kvh, n, dim), device="cuda").bfloat16().transpose(0, 1)
    nat.kv_paged_append(None, k, v, k_cache, v_cache, i32([[4, 2], [0, 3]]), i32([6, 0]))
    for r, (pg, slot) in enumerate([(4, 6), (4, 7), (2, 0), (0, 0), (0, 1), (0, 2)]):
        assert torch.equal(both[pg, 0, :, slot], k[r]) and torch.equal(both[pg, 1, :, slot], v[r])
    assert int((both != 0).sum()) == int((k != 0).sum() + (v != 0).sum())


# ---------------------------------------------------------------- attention

def check_attention(nat, lengths, rows, page, heads, kvh, dim, dtype, *, seed=0, scale=None, spoil=None, hide=True,
                    values=1.0, room=1):
    seen = [max(0, x + rows) for x in lengths]
    k_cache, v_cache, table = ref.make_pages(seen, page, kvh, dim, dtype, seed, extra_cols=-(-room // page))
    v_cache *= values
    if spoil is not None:
        spoil(table)
    if hide:  # NaN and infinities in every slot that nobody sees
        used = torch.zeros(k_cache.shape[:2], dtype=torch.bool)
        for b, n in enumerate(seen):
            for p in range(min(n, table.shape[1] * page)):
                if 0 <= int(table[b, p // page]) < k_cache.shape[0]:
                    used[int(table[b, p // page]), p % page] = True
        k_cache[~used] = float("nan")
        v_cache[~used] = float("inf")
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn((len(lengths), rows, heads, dim), generator=g).to(dtype)
    scale = dim ** -0.5 if scale is None else scale
    want, bound = ref.attention(q, k_cache, v_cache, table, lengths, scale)
    args = (k_cache.cuda(), v_cache.cuda(), table.cuda(), i32(lengths))
    got = nat.kv_paged_attention_decode(q.cuda() if rows > 1 else q[:, 0].cuda(), *args, softmax_scale=scale)
    assert got.dtype == dtype and got.shape == (q.shape if rows > 1 else q[:, 0].shape)
    ref.within(got.reshape(q.shape), want, bound)
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kvh,dim", [(28, 4, 128), (2, 2, 64), (12, 1, 256), (40, 2, 64), (17, 1, 128),
                                           (6, 3, 96), (4, 2, 8), (5, 1, 40), (6, 2, 192), (33, 1, 112), (3, 1, 200)])
@pytest.mark.parametrize("room", [1, 200000])
def test_attention_lengths_and_heads(nat, dtype, heads, kvh, dim, room):
    check_attention(nat, [0, 30, 31, 32, 126, 127, 128, 299, -1, 700], 1, 16, heads, kvh, dim, dtype, seed=dim, room=room)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [2, 3, 5, 8])
@pytest.mark.parametrize("heads,kvh,dim", [(7, 1, 128), (4, 4, 64), (8, 2, 256), (12, 2, 96)])
@pytest.mark.parametrize("longest,room", [(333, 1), (813, 1), (813, 200000)])
def test_attention_of_several_rows(nat, dtype, rows, heads, kvh, dim, longest, room):
    """Of small and of large tables, whose workgroups take 16 and 32 rows and heads."""
    check_attention(nat, [0, 1, 29, 60, 125, -8, longest], rows, 8, heads, kvh, dim, dtype, seed=rows, room=room)


@pytest.mark.parametrize("page", [1, 3, 8, 31, 100, 256, 1024])
def test_attention_page_sizes(nat, page):
    check_attention(nat, [250, 0, 99, 1030], 1, page, 8, 2, 64, torch.float16, seed=page)
    check_attention(nat, [250, 31, 99], 4, page, 4, 2, 64, torch.bfloat16, seed=page)


@pytest.mark.parametrize("sequences,longest", [(1, 9000), (2, 20000), (70, 400), (200, 130)])
def test_attention_splits(nat, sequences, longest):
    """Few long sequences (many splits each) and many of different lengths."""
    lengths = [longest * (b + 1) // sequences - 1 for b in range(sequences)]
    check_attention(nat, lengths, 1, 64, 2, 1, 64, torch.bfloat16, seed=sequences, hide=sequences < 100)


@pytest.mark.parametrize("share", [1, 2])
@pytest.mark.parametrize("dtype,kvh,group,dim,rows", [
    (torch.bfloat16, 64, 1, 64, 1), (torch.float16, 64, 3, 64, 5), (torch.bfloat16, 64, 10, 64, 2),
    (torch.bfloat16, 64, 17, 64, 3), (torch.float16, 32, 4, 128, 1), (torch.bfloat16, 32, 9, 128, 2),
    (torch.float16, 32, 33, 128, 1), (torch.bfloat16, 64, 2, 80, 1), (torch.bfloat16, 16, 3, 256, 1),
    (torch.float16, 16, 2, 256, 4)])
def test_attention_runs_across_sequences(nat, share, dtype, kvh, group, dim, rows):
    """Many heads and enough positions that a workgroup's run goes on from one
    sequence into the next; in whole (share 1) also more than the cache holds,
    so that the values pass it by."""
    lengths = [n // share for n in (5200, 0, 127, 99, -20, 128, 900, 1, 3000)]
    check_attention(nat, lengths, rows, 64, kvh * group, kvh, dim, dtype, seed=dim + rows)


def test_attention_runs_across_many_sequences(nat):
    lengths = [(37 * b) % 190 - 3 for b in range(90)]
    lengths[40] = 9000
    check_attention(nat, lengths, 1, 16, 128, 64, 64, torch.bfloat16, seed=4)
    check_attention(nat, lengths, 2, 16, 64, 32, 128, torch.float16, seed=5)


@pytest.mark.parametrize("rows", [1, 3])
def test_attention_many_sequences_alone(nat, rows):
    """Each sequence is one workgroup's: all short, in tables of any length, and
    so many that the device is full."""
    lengths = [(53 * b) % 400 - 20 for b in range(70)]
    check_attention(nat, lengths, rows, 16, 4, 1, 128, torch.bfloat16, seed=6)
    check_attention(nat, lengths, rows, 16, 4, 1, 128, torch.float16, seed=6, room=2000)
    lengths = [(211 * b) % 1400 - 20 for b in range(40)]
    check_attention(nat, lengths, rows, 16, 16, 8, 64, torch.bfloat16, seed=7)


@pytest.mark.parametrize("kvh,longest", [(1, 3000), (8, 6000), (2, 40)])
def test_attention_of_more_than_512_sequences(nat, kvh, longest):
    lengths = [(7 * b) % 45 - 2 for b in range(620)]
    lengths[570] = longest
    check_attention(nat, lengths, 1, 16, 2 * kvh, kvh, 64, torch.bfloat16, seed=8)
    lengths[570], lengths[2] = 5, longest
    check_attention(nat, lengths, 1, 16, 2 * kvh, kvh, 64, torch.float16, seed=9, room=600)


def test_attention_leaves_out_bad_pages(nat):
    def spoil(table):
        table[0, 1] = -1
        table[0, 3] = 10 ** 6
        table[1, :] = -3          # no page at all: zeros
        table[2, 0] = -1

    got = check_attention(nat, [70, 40, 7, 33], 1, 16, 4, 2, 64, torch.float16, spoil=spoil)
    assert not got[1].any()
    check_attention(nat, [70, 40, 7, 300], 3, 16, 4, 2, 64, torch.bfloat16, spoil=spoil)


def test_attention_rows_do_not_see_what_follows(nat):
    """A later row's own value is NaN or infinite: earlier rows stay finite."""
    for dim, heads in ((128, 4), (64, 4), (256, 2)):
        for last in (32, 63, 64, 200):
            k, v, table = ref.make_pages([last + 4], 16, 2, dim, torch.bfloat16, last)
            for r, bad in ((2, float("nan")), (3, float("inf"))):
                pos = last + r
                v[int(table[0, pos // 16]), pos % 16] = bad
                k[int(table[0, pos // 16]), pos % 16] = float("nan") if r == 3 else 1.0
            q = torch.randn((1, 4, heads, dim), generator=torch.Generator().manual_seed(last)).bfloat16()
            want, bound = ref.attention(q[:, :2], k, v, table, [last], dim ** -0.5)
            got = nat.kv_paged_attention_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32([last])).cpu()
            ref.within(got[:, :2], want, bound)
            assert got[:, 2:].isnan().all()


def test_attention_extreme_scores(nat):
    """Scores far apart (one weight takes all), equal ones, and a negative or zero scale."""
    for scale in (30.0, 0.0, -0.5):
        check_attention(nat, [500, 31], 1, 16, 4, 2, 64, torch.bfloat16, scale=scale)
        check_attention(nat, [500, 31], 2, 16, 4, 2, 64, torch.float16, scale=scale)
    # fp16 weights far below the largest still count: 60000 of 2^-20 each
    n, dim = 60000, 64
    k = torch.zeros((1, n + 1, 1, dim), dtype=torch.float16, device="cuda")
    v = torch.full_like(k, 16.0)
    k[0, 0, 0, 0], v[0, 0] = 20 * math.log(2), 0.0
    q = torch.zeros((1, 1, dim), dtype=torch.float16, device="cuda")
    q[..., 0] = 1.0
    got = nat.kv_paged_attention_decode(q, k, v, i32([[0]]), i32([n]), softmax_scale=1.0)
    first = math.exp(float(k[0, 0, 0, 0]))
    want = torch.full((1, 1, dim), 16.0 * n / (n + first), dtype=torch.float64)
    ref.within(got, want, (4 * ref.HALF[torch.float16]) * want + ref.TINY[torch.float16])


def test_attention_other_orders(nat):
    """Caches [page][head][slot] of one allocation, queries as columns of a wider matrix."""
    n, kvh, page, dim, heads = 2, 2, 16, 64, 6
    both = torch.randn((9, 2, kvh, page, dim), generator=torch.Generator().manual_seed(1)).half()
    table = torch.tensor([[8, 1, 2], [3, 0, 5]], dtype=torch.int32)
    qkv = torch.randn((n, (heads + 4) * dim), generator=torch.Generator().manual_seed(2)).half()
    k, v = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    q = qkv[:, :heads * dim].unflatten(1, (heads, dim))
    want, bound = ref.attention(q[:, None], k, v, table, [40, 17], dim ** -0.5)
    dboth, dq = both.cuda(), qkv.cuda()[:, :heads * dim].unflatten(1, (heads, dim))
    got = nat.kv_paged_attention_decode(dq, dboth[:, 0].transpose(1, 2), dboth[:, 1].transpose(1, 2), table.cuda(),
                                        i32([40, 17]))
    ref.within(got, want[:, 0], bound[:, 0])
    shared = nat.kv_paged_attention_decode(dq[:, :1].expand(n, heads, dim), dboth[:, 0].transpose(1, 2),
                                           dboth[:, 1].transpose(1, 2), table.cuda(), i32([40, 17]))
    ref.within(shared[:, :1], want[:, :1, 0], bound[:, :1, 0])


def test_offsets_past_32_bits(nat):
    """Pages behind the 2^32nd value of a cache that holds keys and values."""
    page, kvh, dim, heads, lengths = 16, 4, 128, 8, [40, 3, -1, 77]
    pages = 2 ** 32 // (page * kvh * dim) + 1000
    both = torch.empty((pages, 2, page, kvh, dim), dtype=torch.bfloat16, device="cuda")
    k, v = both[:, 0], both[:, 1]
    small_k, small_v, small = ref.make_pages([x + 1 for x in lengths], page, kvh, dim, torch.bfloat16, 12)
    at = pages - 1 - 7 * torch.arange(small_k.shape[0])
    k[at], v[at] = small_k.cuda(), small_v.cuda()
    table = torch.where(small >= 0, at[small.clamp(min=0).long()].int(), small)
    g = torch.Generator().manual_seed(13)
    new = torch.randn((4, kvh, dim), generator=g).bfloat16()
    q = torch.randn((4, heads, dim), generator=g).bfloat16()
    got_q = nat.kv_paged_append(q.cuda(), new.cuda(), -new.cuda(), k, v, table.cuda(), i32(lengths))
    for b, n in enumerate(lengths):
        if n >= 0:
            small_k[int(small[b, n // page]), n % page], small_v[int(small[b, n // page]), n % page] = new[b], -new[b]
    assert torch.equal(k[at].cpu(), small_k) and torch.equal(v[at].cpu(), small_v)
    want, bound = ref.attention(q[:, None], small_k, small_v, small, lengths, dim ** -0.5)
    got = nat.kv_paged_attention_decode(got_q, k, v, table.cuda(), i32(lengths))
    ref.within(got, want[:, 0], bound[:, 0])


def test_attention_at_far_positions(nat):
    """A sequence of 2^30 positions of which the last page alone is there."""
    page, dim, far = 2 ** 16, 64, 2 ** 30 + 100
    g = torch.Generator().manual_seed(14)
    k, v = (torch.randn((1, page, 1, dim), generator=g).half() for _ in range(2))
    q = torch.randn((1, 2, dim), generator=g).half()
    table = torch.full((1, far // page + 1), -1, dtype=torch.int32)
    table[0, -1] = 0
    want, bound = ref.attention(q[:, None], k, v, torch.zeros((1, 1), dtype=torch.int32), [100], dim ** -0.5)
    got = nat.kv_paged_attention_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32([far]))
    ref.within(got, want[:, 0], bound[:, 0])


def test_no_sequences(nat):
    cache = torch.zeros((2, 4, 1, 16), dtype=torch.float16, device="cuda")
    none = torch.empty((0, 1, 16), dtype=torch.float16, device="cuda")
    table, lengths = torch.empty((0, 3), dtype=torch.int32, device="cuda"), i32([])
    got = nat.kv_paged_append(none, none, none, cache, cache.clone(), table, lengths)
    assert got.shape == (0, 1, 16)
    assert nat.kv_paged_attention_decode(got, cache, cache.clone(), table, lengths).shape == (0, 1, 16)


def test_attention_the_library_s_own_scratch(nat):
    from pocketlm_amd import _lib

    lib = _lib.load()
    k, v, table = (t.cuda() for t in ref.make_pages([900, 300], 16, 2, 64, torch.bfloat16, 5))
    assert lib.kv_paged_attention_scratch_bytes(2, 1, 4, 2, 64, 16 * table.shape[1]) > 0
    q = torch.randn((2, 4, 64), device="cuda").bfloat16()
    lengths = i32([899, 299])
    want = nat.kv_paged_attention_decode(q, k, v, table, lengths)
    out = torch.zeros_like(q)
    lib.pocketlm_set_stream(torch.cuda.current_stream().cuda_stream)
    assert lib.kv_paged_attention_decode_u16(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), table.data_ptr(), lengths.data_ptr(), out.data_ptr(), None, 0, 2, 1, 4,
        2, 64, 256, 0, 64, table.shape[1], k.shape[0], 16, k.stride(0), k.stride(1), k.stride(2), 0.125, 1) == 0
    assert torch.equal(out, want)


# ---------------------------------------------------------------- a decode step

class Step:
    """A layer's attention part for a batch: norm, q/k/v, append, attention, o."""

    def __init__(self, nat, dtype=torch.bfloat16, sequences=5, hidden=384, heads=6, kvh=2, dim=64, page=16, room=300):
        g = torch.Generator().manual_seed(77)

        def weight(out, cols):
            w = torch.randn((out, cols), generator=g).to(torch.float8_e4m3fn)
            return w.cuda(), (torch.rand(((out + 127) // 128, (cols + 127) // 128), generator=g) * 0.01 + 0.01).cuda()

        self.nat, self.dtype, self.heads, self.kvh, self.dim, self.hidden = nat, dtype, heads, kvh, dim, hidden
        self.qkv, self.o = weight((heads + 2 * kvh) * dim, hidden), weight(hidden, heads * dim)
        self.norm = torch.randn((hidden,), generator=g).to(dtype).cuda()
        k, v, table = ref.make_pages([room] * sequences, page, kvh, dim, dtype, 78)
        self.k, self.v, self.table = k.cuda(), v.cuda(), table.cuda()
        self.freq = nat.kv_rope_frequencies(dim, 1e6)

    def __call__(self, x, residual, lengths):
        nat, heads, kvh, dim = self.nat, self.heads, self.kvh, self.dim
        n, rows = x.shape[:2]
        normed, summed = nat.fp8_e4m3_rms_norm_rows(x, self.norm, rms_eps=1e-6, residual=residual)
        qkv = nat.fp8_e4m3_block_matmul(normed, *self.qkv, out_dtype=self.dtype)
        q, k, v = (t.unflatten(1, (-1, dim)) for t in qkv.split([heads * dim, kvh * dim, kvh * dim], 1))
        q = nat.kv_paged_append(q, k, v, self.k, self.v, self.table, lengths, rope_frequencies=self.freq)
        heads_out = nat.kv_paged_attention_decode(q.view(n, rows, heads, dim), self.k, self.v, self.table, lengths)
        back = nat.fp8_e4m3_quantize_rows(heads_out.view(n * rows, heads * dim))
        out = nat.fp8_e4m3_block_matmul(back, *self.o, out_dtype=self.dtype)
        lengths += rows
        return {"normed": normed, "sum": summed, "qkv": qkv, "q": q, "heads": heads_out, "back": back, "out": out}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 4])
def test_decode_steps_one_after_another(nat, dtype, rows):
    """Each operator's result against its definition on what it was given."""
    step = Step(nat, dtype)
    before = [0, 30, 111, -1, 64]
    lengths = i32(before)
    for i in range(3):
        x, r = (torch.randn((5, rows, step.hidden), generator=torch.Generator().manual_seed(10 * i + j)).to(dtype).cuda()
                for j in (0, 1))
        k_was = step.k.cpu()
        at = [b + i * rows if b >= 0 else -1 for b in before]
        lengths[3] = -1
        s = step(x, r, lengths)
        given = [t.cpu() for t in (*s["normed"], *step.qkv)]
        want, size = ref.matmul(*given)
        ref.within(s["qkv"], want, ref.matmul_bound(want, size, *given, dtype), "qkv")
        qkv = s["qkv"].cpu()
        parts = qkv.split([step.heads * step.dim, step.kvh * step.dim, step.kvh * step.dim], 1)
        q, k, v = (t.unflatten(1, (-1, step.dim)) for t in parts)
        want_k, bound_k = k_was.double(), torch.zeros(k_was.shape, dtype=torch.float64)
        for n, where in enumerate(ref.places(step.table, at, 5 * rows)):
            if where is None:
                assert not s["q"][n].any()
                continue
            b, pos = where
            y, e = ref.rotate(q[n], pos, step.freq.cpu(), False)
            ref.within(s["q"][n], y, e + ref.HALF[dtype] * (y.abs() + e) + ref.TINY[dtype], "q")
            y, e = ref.rotate(k[n], pos, step.freq.cpu(), False)
            slot = (int(step.table[b, pos // 16]), pos % 16)
            want_k[slot], bound_k[slot] = y, e + ref.HALF[dtype] * (y.abs() + e) + ref.TINY[dtype]
            assert torch.equal(step.v[slot].cpu(), v[n])
        ref.within(step.k, want_k, bound_k, "keys")
        want, bound = ref.attention(s["q"].cpu().view(5, rows, step.heads, step.dim), step.k.cpu(), step.v.cpu(),
                                    step.table.cpu(), at, step.dim ** -0.5)
        ref.within(s["heads"], want, bound, "attention")
        given = [t.cpu() for t in (*s["back"], *step.o)]
        want, size = ref.matmul(*given)
        ref.within(s["out"], want, ref.matmul_bound(want, size, *given, dtype), "out")


def test_a_captured_step_follows_its_lengths(nat):
    """One graph of a decode step, replayed with new inputs and growing lengths
    (from one split to several) between eager steps on another cache: each
    replay has the eager step's bits."""
    eager, captured = Step(nat, room=1200), Step(nat, room=1200)
    x = torch.randn((5, 1, eager.hidden), device="cuda").bfloat16()
    r = torch.randn((5, 1, eager.hidden), device="cuda").bfloat16()
    gx, gr, glen = x.clone(), r.clone(), i32([0, 100, 127, -1, 900])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = captured(gx, gr, glen)
    for i, lengths in enumerate(([0, 100, 127, -1, 900], [1, 101, 128, 5, 901], [300, 700, 1100, 0, 2], [40, 40, 40, 40, 40])):
        x = torch.randn((5, 1, eager.hidden), generator=torch.Generator().manual_seed(i)).bfloat16().cuda()
        elen = i32(lengths)
        captured.k.copy_(eager.k)
        captured.v.copy_(eager.v)
        want = eager(x, r, elen)
        gx.copy_(x)
        gr.copy_(r)
        glen.copy_(i32(lengths))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held["out"], want["out"]) and torch.equal(held["heads"], want["heads"])
        assert torch.equal(captured.k, eager.k) and torch.equal(glen, elen)
        torch.randn((64, 64), device="cuda").matmul(torch.randn((64, 64), device="cuda"))


def test_a_captured_attention_follows_its_lengths(nat):
    """One graph over short, ragged, long and idle sequences in turn: each deal
    of the units, from the lengths that the replay finds."""
    sequences, dim = 40, 64
    k, v, table = ref.make_pages([1500] * sequences, 16, 8, dim, torch.bfloat16, 31)
    q = torch.randn((sequences, 16, dim), generator=torch.Generator().manual_seed(32)).bfloat16()
    dk, dv, dtable, dq, lengths = k.cuda(), v.cuda(), table.cuda(), q.cuda(), i32([7] * sequences)
    nat.kv_paged_attention_decode(dq, dk, dv, dtable, lengths)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = nat.kv_paged_attention_decode(dq, dk, dv, dtable, lengths)
    for now in ([9] * sequences, [1499] + [3] * 39, [300 + 30 * b for b in range(40)], [-1] * 39 + [1200],
                [-1] * sequences, [1499] * 3 + [100] * 37, [1400] * sequences):
        lengths.copy_(i32(now))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        want, bound = ref.attention(q[:, None], k, v, table, now, dim ** -0.5)
        ref.within(out, want[:, 0], bound[:, 0])
        assert torch.equal(out, nat.kv_paged_attention_decode(dq, dk, dv, dtable, lengths))


def test_two_captured_graphs_at_once(nat):
    """Two graphs of long attention calls replayed on two streams: neither
    uses the other's scratch."""
    graphs = []
    for seed in (1, 2):
        k, v, table = (t.cuda() for t in ref.make_pages([6000, 5000], 16, 2, 128, torch.bfloat16, seed))
        q = torch.randn((2, 14, 128), generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()
        lengths = i32([5999, 4999])
        want = nat.kv_paged_attention_decode(q, k, v, table, lengths)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = nat.kv_paged_attention_decode(q, k, v, table, lengths)
        graphs.append((graph, out, want, torch.cuda.Stream(), (k, v, table, q, lengths)))
    torch.cuda.synchronize()
    for _ in range(4):
        for graph, out, _w, stream, _keep in graphs:
            with torch.cuda.stream(stream):
                out.zero_()
                graph.replay()
        torch.cuda.synchronize()
        for _g, out, want, _s, _keep in graphs:
            assert torch.equal(out, want)


def test_calls_on_another_stream(nat):
    step, other = Step(nat), Step(nat)
    x = torch.randn((5, 1, step.hidden), device="cuda").bfloat16()
    want = step(x, x, i32([3, 4, 5, 6, 7]))
    lengths = i32([3, 4, 5, 6, 7])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = other(x, x, lengths)
    stream.synchronize()
    assert torch.equal(got["out"], want["out"]) and torch.equal(other.k, step.k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("room", [1, 200000])
def test_attention_of_scores_past_2_to_the_24(nat, dtype, room):
    """Scores that fp32 holds in steps of whole numbers, exact ones: 2^15 apart
    at least, so the largest position's value is the result."""
    n, dim, page = 40, 64, 16
    lengths = [20 + 13 * b for b in range(n)]
    k, v, table = ref.make_pages([x + 1 for x in lengths], page, 1, dim, dtype, 41, extra_cols=-(-room // page))
    k.zero_()
    want = torch.zeros((n, 2, dim), dtype=dtype)
    for b, length in enumerate(lengths):
        for p in range(length + 1):
            k[int(table[b, p // page]), p % page, 0, :8] = p % 97
        at = (7 * b) % (length + 1)
        slot = (int(table[b, at // page]), at % page, 0)
        k[slot][:8] = 128 + 3 * b
        want[b, :] = v[slot]
    q = torch.zeros((n, 2, dim), dtype=dtype)
    q[..., :8] = 2.0 ** 15
    got = nat.kv_paged_attention_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32(lengths), softmax_scale=1.0)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 4])
@pytest.mark.parametrize("heads,kvh,dim", [(28, 4, 128), (8, 8, 64), (4, 2, 256), (6, 3, 96)])
def test_attention_weights_keep_more_bits_than_the_cache(nat, dtype, rows, heads, kvh, dim):
    """The bound of ref.attention with 2^-15 (fp16 2^-21, and 2^-38 of the row's largest) for a
    weight's rounding: a weight is a value of the cache's type, cut off (2^-7 of it, fp16 2^-10),
    and the rest in that type, rounded (2^-8 of the rest, fp16 2^-11)."""
    lengths = [600, 17, 1200]
    k, v, table = ref.make_pages([x + rows for x in lengths], 16, kvh, dim, dtype, 51)
    q = torch.randn((3, rows, heads, dim), generator=torch.Generator().manual_seed(52)).to(dtype)
    want, _ = ref.attention(q, k, v, table, lengths, dim ** -0.5)
    bound = torch.zeros_like(want)
    for b, length in enumerate(lengths):
        for r in range(rows):
            at = torch.arange(length + r + 1)
            page, slot = table[b][at // 16].long(), at % 16
            for h in range(kvh):
                group = slice(h * (heads // kvh), (h + 1) * (heads // kvh))
                ks, vs, qs = k[page, slot, h].double(), v[page, slot, h].double().abs(), q[b, r, group].double()
                off = (qs.abs() @ ks.abs().t()) * dim ** -0.5 * (dim + 4) * 2.0 ** -23
                p = torch.softmax(qs @ ks.t() * dim ** -0.5, dim=1)
                share = 2 * off + 2.0 ** -20 + (len(at) / 32 + 64) * 2.0 ** -23
                weight = 2.0 ** -15 * p if dtype == torch.bfloat16 else 2.0 ** -21 * p + 2.0 ** -38 * p.amax(1, keepdim=True)
                wide = (p * share + weight) @ vs + share.amax(1, keepdim=True) * (p @ vs)
                o = want[b, r, group].abs()
                bound[b, r, group] = wide + ref.HALF[dtype] * (o + wide) + ref.TINY[dtype]
    got = nat.kv_paged_attention_decode(q.cuda() if rows > 1 else q[:, 0].cuda(), k.cuda(), v.cuda(), table.cuda(),
                                        i32(lengths))
    ref.within(got.reshape(q.shape), want, bound)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_of_infinite_values_that_are_seen(nat, dtype):
    """An infinite value with a weight above 0 is the result's, with its sign; equal weights are 1."""
    k, v, table = ref.make_pages([300, 300, 40], 16, 2, 64, dtype, 53)
    for b, (pos, sign) in enumerate(((200, 1), (3, -1), (39, 1))):
        v[int(table[b, pos // 16]), pos % 16] = sign * float("inf")
    q = torch.randn((3, 4, 64), generator=torch.Generator().manual_seed(54)).to(dtype)
    q[2] = 0.0
    got = nat.kv_paged_attention_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), i32([299, 299, 39])).cpu()
    assert torch.equal(got[0], torch.full_like(got[0], float("inf")))
    assert torch.equal(got[1], torch.full_like(got[1], -float("inf")))
    assert torch.equal(got[2], torch.full_like(got[2], float("inf")))


@pytest.mark.parametrize("sequences,longest,kvh", [(1, 9000, 2), (40, 3000, 2), (300, 1500, 8), (90, 9000, 64), (1200, 700, 1)])
def test_attention_writes_within_its_scratch(nat, sequences, longest, kvh):
    """The C entry with as much scratch as it asks for, at the end of a buffer whose front and back stay as they are."""
    from pocketlm_amd import _lib

    lib, dim, page, guard = _lib.load(), 64, 16, 1 << 20
    lengths = [(97 * b) % 190 - 3 for b in range(sequences)]
    lengths[sequences // 2] = longest
    k, v, table = (t.cuda() for t in ref.make_pages([max(0, x + 1) for x in lengths], page, kvh, dim, torch.float16, 61))
    q = torch.randn((sequences, 2 * kvh, dim), generator=torch.Generator().manual_seed(62)).half().cuda()
    dl = i32(lengths)
    need = lib.kv_paged_attention_scratch_bytes(sequences, 1, 2 * kvh, kvh, dim, page * table.shape[1])
    assert need > 0 and need % 8 == 0
    room = torch.full((2 * guard + need,), 0xA5, dtype=torch.uint8, device="cuda")
    out = torch.zeros_like(q)
    lib.pocketlm_set_stream(torch.cuda.current_stream().cuda_stream)
    assert lib.kv_paged_attention_decode_u16(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), table.data_ptr(), dl.data_ptr(), out.data_ptr(), room.data_ptr() + guard,
        need, sequences, 1, 2 * kvh, kvh, dim, 2 * kvh * dim, 0, dim, table.shape[1], k.shape[0], page, k.stride(0),
        k.stride(1), k.stride(2), 0.125, 0) == 0
    assert torch.equal(out, nat.kv_paged_attention_decode(q, k, v, table, dl))
    assert bool((room[:guard] == 0xA5).all()) and bool((room[guard + need:] == 0xA5).all())


@pytest.mark.parametrize("interleaved", [False, True])
def test_append_far_positions_store_their_keys(nat, interleaved):
    """Keys and values of a position beyond 2^30, in caches of their own whose pages share one row."""
    dim, far, page = 64, 2 ** 30 + 12345, 2 ** 20
    rows = [torch.zeros((1, 1, 1, dim), dtype=torch.float16, device="cuda") for _ in range(2)]
    k_cache, v_cache = (t.expand(1, page, 1, dim) for t in rows)
    freq = nat.kv_rope_frequencies(dim, 1e6)
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn((1, 1, dim), generator=g).half() for _ in range(2))
    table = torch.zeros((1, 2 ** 10 + 1), dtype=torch.int32, device="cuda")
    nat.kv_paged_append(None, k.cuda(), v.cuda(), k_cache, v_cache, table, i32([far]), rope_frequencies=freq,
                        interleaved=interleaved)
    want, bound = ref.rotate(k[0], far, freq.cpu(), interleaved)
    ref.within(rows[0][0, 0], want, bound + ref.HALF[torch.float16] * (want.abs() + bound) + ref.TINY[torch.float16])
    assert torch.equal(rows[1][0].cpu(), v)


def test_captured_steps_with_an_idle_sequence(nat):
    """The step with the lengths of live sequences advanced behind it, captured
    once and replayed for five tokens: an idle sequence stays idle."""
    eager, captured = Step(nat), Step(nat)
    captured.k.copy_(eager.k)
    captured.v.copy_(eager.v)

    def step(of, x, lengths):
        out = of(x, x, lengths.clone())
        lengths += lengths >= 0
        return out["out"]

    x = torch.randn((5, 1, eager.hidden), generator=torch.Generator().manual_seed(71)).bfloat16().cuda()
    lengths, glen, gx = i32([0, 100, -1, 31, 127]), i32([0, 100, -1, 31, 127]), x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(captured, gx, glen)
    for i in range(5):
        want = step(eager, x, lengths)
        gx.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want) and torch.equal(captured.k, eager.k) and torch.equal(captured.v, eager.v)
        assert lengths.tolist() == glen.tolist() == [i + 1, 101 + i, -1, 32 + i, 128 + i]
        x = torch.randn((5, 1, eager.hidden), generator=torch.Generator().manual_seed(72 + i)).bfloat16().cuda()
