"""Decode steps over e4m3 pages that are large enough for the launch's other
choices (values read past the caches, a third workgroup to a compute unit),
against the definition in 64 bits.  Tables repeat a small pool's pages."""

from __future__ import annotations

import pytest
import torch

import paged_refs as pref

pytestmark = pytest.mark.gpu

BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
POOL = 300


@pytest.fixture(scope="module")
def nat():
    from pocketlm_amd import native

    assert native.native_paged_kv_available(), "libpocketlm_hip.so must load"
    return native


def made(lengths, rows, page, heads, kvh, dim, dtype, seed):
    """(q, caches, scales, table, lengths): tables of random pages of the pool, wide enough for every sequence."""
    caches, scales, _ = pref.make_pages([POOL * page], page, kvh, dim, E4M3, seed, spare=0)
    g = torch.Generator().manual_seed(seed + 1)
    cols = (max(lengths) + rows + page - 1) // page + 3
    table = torch.randint(0, POOL, (len(lengths), cols), generator=g, dtype=torch.int32)
    q = torch.randn((len(lengths), rows, heads, dim), generator=g).to(dtype).cuda()
    return q, caches, scales, table, torch.tensor(lengths, dtype=torch.int32, device="cuda")


def definition(q, caches, scales, table, lengths):
    n, rows, dim = q.shape[0], q.shape[1], q.shape[3]
    # weights in two bf16 halves: 15 bits of each
    want, bound = pref.chunk(q.flatten(0, 1), *caches, table, lengths.tolist(), [rows * b for b in range(n + 1)], dim ** -0.5,
                             scales=scales, weight=2.0 ** -15)
    return want.view(q.shape), bound.view(q.shape)


def ragged(count, total, longest):
    """`count` lengths that sum to about `total`, the first `longest`, one of 0 and one idle among them."""
    rest = (total - longest) // (count - 3)
    return [longest, 0, -1, *(rest - 700 + 1400 * b // (count - 3) for b in range(count - 3))]


# (units of 128 positions: from 1024 on, at 4 heads of 128, values are read past the caches, from 2048 on workgroups are
# three to a compute unit; heads of 64 are always read through the caches)
@pytest.mark.parametrize("heads,kvh,dim,rows,dtype", [(28, 4, 128, 1, BF16), (28, 4, 128, 2, F16), (12, 4, 128, 3, BF16),
                                                      (16, 8, 64, 1, BF16), (32, 8, 64, 4, F16), (20, 10, 48, 1, BF16)])
@pytest.mark.parametrize("units,longest", [(2200, 60000), (1400, 40000), (2200, 12000)])
def test_large_batches(nat, heads, kvh, dim, rows, dtype, units, longest):
    units = units * 512 // (kvh * dim)
    lengths = ragged(26, 128 * units, longest)
    q, caches, scales, table, on_device = made(lengths, rows, 16, heads, kvh, dim, dtype, dim + rows)
    got = nat.kv_paged_attention_decode_e4m3(q[:, 0] if rows == 1 else q, *caches, *scales, table.cuda(), on_device)
    want, bound = definition(q, caches, scales, table, on_device)
    pref.agree(got.view(want.shape), want, bound)


@pytest.mark.parametrize("heads,kvh,dim", [(28, 4, 128), (16, 8, 64)])
@pytest.mark.parametrize("scratch", ["caller's", "library's"])
def test_scratch_of_a_large_batch(nat, heads, kvh, dim, scratch):
    """Stays within kv_paged_attention_scratch_bytes, also where the largest number of runs is taken; the largest table
    with small lengths, and the other way round, in the same scratch."""
    from pocketlm_amd import _lib

    lib = _lib.load()
    page = 16
    lengths = ragged(26, 128 * 2200 * 512 // (kvh * dim), 60000)
    q, caches, scales, table, on_device = made(lengths, 1, page, heads, kvh, dim, BF16, 3)
    table_d, q = table.cuda(), q[:, 0].contiguous()
    need = lib.kv_paged_attention_scratch_bytes(len(lengths), 1, heads, kvh, dim, table.shape[1] * page)
    assert need > 0
    held = torch.full((need + (1 << 20),), 0xA5, dtype=torch.uint8, device="cuda")
    for values in (on_device, on_device // 100, torch.full_like(on_device, int(on_device.max())), on_device):
        want = nat.kv_paged_attention_decode_e4m3(q, *caches, *scales, table_d, values)
        out = torch.zeros_like(q)
        lib.pocketlm_set_stream(torch.cuda.current_stream().cuda_stream)
        code = lib.kv_paged_attention_decode_e4m3(
            q.data_ptr(), caches[0].data_ptr(), caches[1].data_ptr(), scales[0].data_ptr(), scales[1].data_ptr(),
            table_d.data_ptr(), values.data_ptr(), out.data_ptr(), held.data_ptr() if scratch == "caller's" else None,
            need if scratch == "caller's" else 0, len(lengths), 1, heads, kvh, dim, heads * dim, 0, dim, table.shape[1], POOL,
            page, *caches[0].stride()[:3], *scales[0].stride()[:2], dim ** -0.5, 1)
        assert code == 0
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert bool((held[need:] == 0xA5).all())


def test_a_large_batch_in_a_graph(nat):
    """Captured where the lengths are short, replayed where they take other launches' shapes."""
    heads, kvh, dim = 28, 4, 128
    lengths = ragged(26, 128 * 2200, 60000)
    q, caches, scales, table, on_device = made(lengths, 1, 16, heads, kvh, dim, BF16, 5)
    q, table_d, many = q[:, 0], table.cuda(), on_device.clone()
    on_device.fill_(100)
    nat.kv_paged_attention_decode_e4m3(q, *caches, *scales, table_d, on_device)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = nat.kv_paged_attention_decode_e4m3(q, *caches, *scales, table_d, on_device)
    for values in (many, many // 2, torch.full_like(many, 90), many, torch.full_like(many, -1), many):
        on_device.copy_(values)
        want = nat.kv_paged_attention_decode_e4m3(q, *caches, *scales, table_d, on_device)
        torch.cuda.synchronize()
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
