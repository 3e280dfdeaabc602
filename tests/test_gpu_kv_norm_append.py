"""Appends to a paged cache that norm queries and keys, and appends to e4m3
pages, against the definitions in 64 bits."""

from __future__ import annotations

import pytest
import torch

import batched_refs as ref
import paged_refs as pref

pytestmark = pytest.mark.gpu

EPS = 1e-6
DTYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def nat():
    from pocketlm_amd import native

    assert native.native_paged_kv_available(), "libpocketlm_hip.so must load on the GPU box"
    return native


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def check(nat, e4m3, lengths, rows, page, heads, kvh, dim, dtype, *, pairs=None, interleaved=False, norms=True, starts=None,
          eps=EPS, seed=0, spoil=None, make=None):
    """One append into caches that hold values everywhere; every slot is compared."""
    total = sum(rows) if starts is None else starts[-1]
    behind = 3 if starts is not None else 0
    g = torch.Generator().manual_seed(seed)
    lens = [max(0, x) + r for x, r in zip(lengths, rows)]
    (dk, dv), (ks, vs), table = pref.make_pages(lens, page, kvh, dim, torch.float8_e4m3fn if e4m3 else dtype, seed)
    if spoil is not None:
        spoil(table)
    qkv = torch.randn((total + behind, (heads + 2 * kvh) * dim), generator=g).to(dtype)
    if make is not None:
        make(qkv)
    q, k, v = (t.unflatten(1, (-1, dim)) for t in qkv.split([heads * dim, kvh * dim, kvh * dim], 1))
    wq = (1 + 0.2 * torch.randn(dim, generator=g)).to(dtype) if norms else None
    wk = (1 + 0.2 * torch.randn(dim, generator=g)).to(dtype) if norms else None
    pairs = dim // 2 if pairs is None else pairs
    freq = torch.tensor([1e4 ** (-i / max(1, pairs)) for i in range(pairs)], dtype=torch.float64)
    want_k, want_v = (t.view(torch.uint8).cpu() if e4m3 else t.cpu() for t in (dk, dv))
    want_k, want_v = want_k.clone(), want_v.clone()
    old_ks, old_vs = (ks.cpu(), vs.cpu()) if e4m3 else (None, None)
    rejected = i32([5])
    gq, gk, gv = (t.unflatten(1, (-1, dim)) for t in qkv.cuda().split([heads * dim, kvh * dim, kvh * dim], 1))
    kw = dict(rms_eps=eps, row_starts=None if starts is None else i32(starts), rope_frequencies=freq.cuda() if pairs else None,
              interleaved=interleaved, rejected=rejected)
    weights = [None if w is None else w.cuda() for w in (wq, wk)]
    if e4m3:
        got = nat.kv_paged_append_e4m3(gq if heads else None, gk, gv, dk, dv, ks, vs, table.cuda(), i32(lengths),
                                       q_norm_weight=weights[0], k_norm_weight=weights[1], **kw)
    else:
        got = nat.kv_paged_norm_append(gq if heads else None, gk, gv, *weights, dk, dv, table.cuda(), i32(lengths), **kw)
    want_q, bound_q = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    touched = torch.zeros(want_k.shape[:2], dtype=torch.bool)
    refused = 0
    held = {}
    for r, where in enumerate(ref.places(table, lengths, total + behind, starts)):
        if where is None:
            continue
        b, pos = where
        if heads:
            z, off = pref.normed_rotated(q[r], wq, eps, pos, freq, interleaved)
            plain = not norms and not pairs
            want_q[r], bound_q[r] = z, off + (0 if plain else ref.HALF[dtype] * (z.abs() + off) + ref.TINY[dtype])
        index = pos // page
        pid = int(table[b, index]) if index < table.shape[1] else -1
        if not 0 <= pid < want_k.shape[0]:
            refused += 1
            continue
        touched[pid, pos % page] = True
        held[pid, pos % page] = (r, *pref.normed_rotated(k[r], wk, eps, pos, freq, interleaved))
    if heads:
        pref.agree(got.cpu(), want_q, bound_q, "queries")
    else:
        assert got is None
    assert int(rejected) == 5 + refused
    got_k, got_v = (t.view(torch.uint8).cpu() if e4m3 else t.cpu() for t in (dk, dv))
    bits = (lambda t: t) if e4m3 else (lambda t: t.view(torch.int16))
    for t, w in ((got_k, want_k), (got_v, want_v)):
        assert torch.equal(bits(t)[~touched], bits(w)[~touched]), "slots that no row has"
    if e4m3:
        for s, old in ((ks.cpu(), old_ks), (vs.cpu(), old_vs)):
            assert torch.equal(s.transpose(1, 2)[~touched], old.transpose(1, 2)[~touched])
    if not held:
        return refused
    places = list(held)
    pid, slot = torch.tensor([p for p, _ in places]), torch.tensor([s for _, s in places])
    z = torch.stack([held[p][1] for p in places])
    off = torch.stack([held[p][2] for p in places])
    values = torch.stack([v[held[p][0]] for p in places])
    if not e4m3:
        plain = not norms and not pairs
        pref.agree(got_k[pid, slot], z, off + (0 if plain else ref.HALF[dtype] * (z.abs() + off) + ref.TINY[dtype]), "keys")
        assert torch.equal(bits(got_v[pid, slot]), bits(values))
        return refused
    for name, z, off, cache, s in (("keys", z, off, got_k, ks), ("values", values.double(), torch.zeros_like(z), got_v, vs)):
        u, scale, bound, scale_off = pref.quantized(z, off)
        got_scale = s.cpu()[pid, :, slot]
        bad = ~z.isfinite().all(-1)
        assert bool(got_scale[bad].isnan().all()) and bool((cache[pid, slot][bad] == 0x7F).all())
        pref.agree(got_scale[~bad], scale[~bad], scale_off[~bad], name + "' scales")
        pref.agree(cache[pid, slot].view(torch.float8_e4m3fn).double()[~bad], u[~bad], bound[~bad], name)
    return refused


SHAPES = [(28, 4, 128, None, False), (4, 4, 64, None, True), (6, 1, 256, None, False), (5, 5, 96, None, True),
          (8, 2, 128, 32, False), (8, 2, 64, 7, True), (8, 2, 64, 5, False), (4, 4, 80, 0, False), (2, 1, 48, None, False),
          (3, 3, 16, None, True), (0, 2, 128, None, False), (32, 8, 128, 16, True), (2, 2, 240, 120, False)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kvh,dim,pairs,interleaved", SHAPES + [(3, 3, 8, None, False), (4, 2, 40, None, False),
                                                                      (4, 2, 72, None, True), (4, 4, 24, 0, False),
                                                                      (2, 1, 248, 31, False)])
def test_norm_append(nat, dtype, heads, kvh, dim, pairs, interleaved):
    for rows in (1, 3):
        check(nat, False, [0, 17, -1, 403], [rows] * 4, 16, heads, kvh, dim, dtype, pairs=pairs, interleaved=interleaved,
              seed=rows)


@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kvh,dim,pairs,interleaved", SHAPES)
def test_append_e4m3(nat, dtype, norms, heads, kvh, dim, pairs, interleaved):
    for rows in (1, 3):
        check(nat, True, [0, 17, -1, 403], [rows] * 4, 16, heads, kvh, dim, dtype, pairs=pairs, interleaved=interleaved,
              norms=norms, seed=rows)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("page", [1, 5, 64])
def test_prompts_of_ragged_lengths(nat, e4m3, page):
    """Sequences without rows, idle ones, and rows behind the last sequence."""
    rows = [40, 0, 1, 77, 9, 0]
    starts = [sum(rows[:i]) for i in range(7)]
    check(nat, e4m3, [0, 3, 31, 0, -2, 8], rows, page, 4, 2, 64, torch.bfloat16, starts=starts, seed=page)


@pytest.mark.parametrize("e4m3,dim,total", [(False, 16, 8400), (True, 16, 8400), (False, 24, 2500), (True, 48, 5003)])
def test_many_rows(nat, e4m3, dim, total):
    """Calls whose workgroups take several rows, across the borders of many short
    sequences, idle ones and ones without rows, and of a long one."""
    rows = [(7 * i) % 23 for i in range(90)]
    rows.append(total - sum(rows))
    lengths = [-1 if i % 13 == 5 else (31 * i) % 40 for i in range(91)]
    starts = [sum(rows[:i]) for i in range(92)]

    def spoil(table):
        table[3] = -1
        table[90, 7] = 10 ** 6

    assert check(nat, e4m3, lengths, rows, 16, 2, 1, dim, torch.bfloat16, starts=starts, seed=dim, spoil=spoil) > 0


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim,interleaved", [(48, False), (48, True), (80, False), (96, True), (208, False), (240, False)])
def test_heads_with_lanes_to_spare_after_nan_in_lds(nat, e4m3, dim, interleaved):
    """Head sizes that leave lanes without values, whose angles nobody wrote: what an attention over NaN left in LDS
    must not reach the head's maximum."""
    pages = torch.full((64, 64, 4, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
    table = torch.arange(64, dtype=torch.int32, device="cuda")[None]
    q = torch.ones((4096, 4, 128), dtype=torch.bfloat16, device="cuda")
    nat.kv_paged_attention_chunk(q, pages, pages, table, i32([0]), i32([0, 4096]))
    check(nat, e4m3, [0, 17, -1, 403], [40, 900, 3, 300], 16, 4, 2, dim, torch.bfloat16, interleaved=interleaved,
          starts=[0, 40, 940, 943, 1243], seed=dim)


@pytest.mark.parametrize("e4m3", [False, True])
def test_rows_without_a_page(nat, e4m3):
    def spoil(table):
        table[0, 0] = -1
        table[1, 0] = 10 ** 6

    refused = check(nat, e4m3, [0, 2, 30], [4, 4, 4], 16, 4, 2, 64, torch.float16, spoil=spoil)
    assert refused == 8
    check(nat, e4m3, [0, 31], [4, 100], 16, 2, 2, 64, torch.float16, starts=[0, 4, 104],
          spoil=lambda table: table.__setitem__((1, slice(3, None)), -1))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** 70, 2.0 ** -80, 0.0])
def test_norms_of_heads_beyond_fp32_squares(nat, e4m3, dtype, size):
    """Heads whose squares leave fp32, or vanish, with an eps that does not hide them."""
    if dtype == torch.float16 and not 2.0 ** -24 < size < 2.0 ** 10:
        size = {2.0 ** 70: 6e3, 2.0 ** -80: 2.0 ** -20}.get(size, size)
    eps = 1e-30 if size > 0 else 1e-6

    def make(qkv):
        qkv.mul_(size)

    check(nat, e4m3, [3, 9], [2, 2], 16, 4, 2, 128, dtype, eps=eps, make=make)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norms", [False, True])
def test_e4m3_heads_of_infinities_zeros_and_small_values(nat, dtype, norms):
    def make(qkv):
        heads = qkv.view(qkv.shape[0], -1, 64)
        heads[0, 4] = 0.0                      # a key of zeros
        heads[1, 5, 3] = float("inf")          # a key with an infinity
        heads[2, 6, 63] = float("nan")         # a value with a NaN
        heads[3, 7] *= 2.0 ** -14 if dtype == torch.float16 else 2.0 ** -130

    check(nat, True, [3], [4], 16, 4, 2, 64, dtype, norms=norms, make=make)


def test_values_on_a_border_of_e4m3(nat):
    """Values halfway between two e4m3 values under a scale of exactly 2^-3: ties go to even bytes."""
    dim = 64
    steps = torch.tensor([17.0, 19, 21, 23, 25, 27, 29, 31, 34, 38, 42, 46, 50, 54, 58, 62])  # halves of 2 and 4 apart
    x = torch.zeros((1, 1, dim))
    x[0, 0, :16] = steps / 8
    x[0, 0, 16] = 448.0 / 8
    x = x.to(torch.bfloat16)
    (dk, dv), (ks, vs), table = pref.make_pages([1], 4, 1, dim, torch.float8_e4m3fn, 0)
    nat.kv_paged_append_e4m3(None, x.cuda(), x.cuda(), dk, dv, ks, vs, table.cuda(), i32([0]))
    page = int(table[0, 0])
    for cache, s in ((dk, ks), (dv, vs)):
        assert float(s[page, 0, 0]) == 0.125
        got = cache.view(torch.uint8)[page, 0, 0].view(torch.float8_e4m3fn).double().cpu()
        want = (x[0, 0].double() * 8).to(torch.float32).to(torch.float8_e4m3fn).double()
        assert torch.equal(got, want)


@pytest.mark.parametrize("e4m3", [False, True])
def test_other_orders_and_strides(nat, e4m3):
    """[page][head][slot] caches, scales with a page stride of their own, rows of odd strides: the same bits."""
    kvh, dim, page, dtype = 2, 64, 8, torch.bfloat16
    lengths, rows = [5, 0], [3, 3]
    lens = [8, 3]
    (dk, dv), (ks, vs), table = pref.make_pages(lens, page, kvh, dim, torch.float8_e4m3fn if e4m3 else dtype, 1)
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn((6, h, dim), generator=g).to(dtype).cuda() for h in (4, kvh, kvh))
    w = (1 + 0.1 * torch.randn(2 * dim, generator=g)).to(dtype).cuda()
    freq = nat.kv_rope_frequencies(dim, 1e4)

    def call(dk, dv, ks, vs, q, k, v, w0, w1):
        kw = dict(rms_eps=EPS, rope_frequencies=freq)
        if e4m3:
            return nat.kv_paged_append_e4m3(q, k, v, dk, dv, ks, vs, table.cuda(), i32(lengths), q_norm_weight=w0,
                                            k_norm_weight=w1, **kw)
        return nat.kv_paged_norm_append(q, k, v, w0, w1, dk, dv, table.cuda(), i32(lengths), **kw)

    raw = (lambda t: t.view(torch.uint8)) if e4m3 else (lambda t: t.view(torch.int16))
    turned = [raw(t).permute(0, 2, 1, 3).contiguous().view(t.dtype).permute(0, 2, 1, 3) for t in (dk, dv)]
    wide = [None, None]
    if e4m3:
        wide = [torch.full((s.shape[0], 3, kvh, page), 7.0, device="cuda")[:, 1] for s in (ks, vs)]
        for t, s in zip(wide, (ks, vs)):
            t.copy_(s)
    odd = [torch.randn((6, 7, dim + 4), generator=g).to(dtype).cuda()[:, :t.shape[1], 1:dim + 1] for t in (q, k, v)]
    for t, s in zip(odd, (q, k, v)):
        t.copy_(s)
    first = call(dk, dv, ks, vs, q, k, v, w[:dim], w[dim:])
    w_odd = torch.empty(2 * dim + 1, dtype=dtype, device="cuda")
    w_odd[1:] = w
    second = call(*turned, *wide, *odd, w_odd[1:dim + 1], w_odd[dim + 1:])
    assert torch.equal(first.view(torch.int16), second.view(torch.int16))
    for a, b in zip((dk, dv), turned):
        assert torch.equal(raw(a).contiguous(), raw(b.contiguous() if not e4m3 else b.view(torch.uint8).contiguous()))
    if e4m3:
        for a, b in zip((ks, vs), wide):
            assert torch.equal(a, b)


def test_without_weights_an_e4m3_append_quantizes_what_the_16_bit_one_rounds(nat):
    """The same rotation: the 16-bit cache's keys are the e4m3 cache's within both roundings."""
    kvh, dim, page, dtype = 4, 128, 16, torch.bfloat16
    lens = [300, 20]
    starts = i32([0, 300, 320])
    (dk, dv), _, table = pref.make_pages(lens, page, kvh, dim, dtype, 1)
    (ek, ev), (ks, vs), _ = pref.make_pages(lens, page, kvh, dim, torch.float8_e4m3fn, 1)
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn((320, h, dim), generator=g).to(dtype).cuda() for h in (8, kvh, kvh))
    freq = nat.kv_rope_frequencies(dim, 1e6)
    table = table.cuda()
    a = nat.kv_paged_append(q, k, v, dk, dv, table, i32([0, 0]), row_starts=starts, rope_frequencies=freq)
    b = nat.kv_paged_append_e4m3(q, k, v, ek, ev, ks, vs, table, i32([0, 0]), row_starts=starts, rope_frequencies=freq)
    assert torch.equal(a, b)
    for s, n in ((0, 300), (1, 20)):
        for c16, c8, scale in ((dk, ek, ks), (dv, ev, vs)):
            x, _ = pref.gathered(c16, None, table[s], n)
            y, _ = pref.gathered(c8, scale, table[s], n)
            top = x.abs().amax(-1, keepdim=True)
            # half a step of e4m3 at the largest value, 2^-4 of it, and the 16-bit rounding
            assert bool(((x - y).abs() <= (2.0 ** -4 + 2.0 ** -8) * x.abs() + 2.0 ** -9 * top / 448 + 2.0 ** -8 * x.abs()).all())


@pytest.mark.parametrize("size", [1.0, 2.0 ** 70])
def test_e4m3_norms_of_queries_or_keys_alone(nat, size):
    """A weight norms its own heads: the rest is as without any, also where a head's squares leave fp32."""
    kvh, dim, page, dtype = 2, 128, 16, torch.bfloat16
    g = torch.Generator().manual_seed(3)
    q, k, v = ((torch.randn((40, h, dim), generator=g) * size).to(dtype).cuda() for h in (6, kvh, kvh))
    w = (1 + 0.2 * torch.randn(dim, generator=g)).to(dtype).cuda()
    freq = nat.kv_rope_frequencies(dim, 1e6)
    starts, lengths = i32([0, 33, 40]), i32([5, 0])

    def run(wq, wk):
        caches, scales, table = pref.make_pages([38, 7], page, kvh, dim, torch.float8_e4m3fn, 1)
        out = nat.kv_paged_append_e4m3(q, k, v, *caches, *scales, table.cuda(), lengths, q_norm_weight=wq, k_norm_weight=wk,
                                       rms_eps=EPS, row_starts=starts, rope_frequencies=freq)
        return [out] + [t.view(torch.uint8) if t.dtype != torch.float32 else t.view(torch.int32) for t in (*caches, *scales)]

    none, both, queries, keys = run(None, None), run(w, w), run(w, None), run(None, w)
    assert torch.equal(queries[0], both[0]) and torch.equal(keys[0], none[0])
    for i in (1, 3):  # keys and their scales
        assert torch.equal(queries[i], none[i]) and torch.equal(keys[i], both[i])
    for i in (2, 4):
        assert all(torch.equal(x[i], none[i]) for x in (both, queries, keys))


def test_an_empty_call(nat):
    (dk, dv), (ks, vs), table = pref.make_pages([4], 4, 1, 64, torch.float8_e4m3fn, 0)
    x = torch.empty((0, 1, 64), dtype=torch.float16, device="cuda")
    assert nat.kv_paged_append_e4m3(x, x, x, dk, dv, ks, vs, table.cuda(), i32([0])).shape == (0, 1, 64)
