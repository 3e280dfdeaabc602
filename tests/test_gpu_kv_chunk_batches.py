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
