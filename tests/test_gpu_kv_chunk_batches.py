"""Attention of chunks where a batch, its values or its weights are uneven."""

from __future__ import annotations

import pytest
import torch

import paged_refs as pref

pytestmark = pytest.mark.gpu

BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def nat():
    from pocketlm_amd import native

    assert native.native_paged_kv_available(), "libpocketlm_hip.so must load on the GPU box"
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
