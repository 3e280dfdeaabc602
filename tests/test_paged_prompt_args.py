"""What the operators over prompts and e4m3 pages refuse, on the CPU: the C
entry points' codes, and the exceptions of the Python calls."""

from __future__ import annotations

import ctypes

import pytest
import torch

from pocketlm_amd import _lib, native


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        from pocketlm_amd import build

        build.build()
    return _lib.load()


A = ctypes.c_void_p(4096)    # an aligned address that is never read
ODD = ctypes.c_void_p(4098)
N = ctypes.c_void_p(0)


def append(lib, e4m3, q=A, k=A, v=A, wq=A, wk=A, q_out=A, kc=A, vc=A, ks=A, vs=A, table=A, lengths=A, starts=N, freq=A,
           rejected=N, rows=2, seqs=2, heads=4, kvh=2, dim=64, pairs=32, inter=0, strides=(256, 64, 128, 64, 128, 64),
           cols=4, pages=8, page=16, cache=(2048, 128, 64), scale=(32, 16), eps=1e-6, code=1):
    if e4m3:
        return lib.kv_paged_append_e4m3(q, k, v, wq, wk, q_out, kc, vc, ks, vs, table, lengths, starts, freq, rejected, rows,
                                        seqs, heads, kvh, dim, pairs, inter, *strides, cols, pages, page, *cache, *scale, eps,
                                        code)
    return lib.kv_paged_norm_append_u16(q, k, v, wq, wk, q_out, kc, vc, table, lengths, starts, freq, rejected, rows, seqs,
                                        heads, kvh, dim, pairs, inter, *strides, cols, pages, page, *cache, eps, code)


@pytest.mark.parametrize("e4m3", [False, True])
def test_append_codes(lib, e4m3):
    names = ["q", "k", "v", "q_out", "kc", "vc", "table", "lengths", "freq"] + (["ks", "vs"] if e4m3 else ["wq", "wk"])
    for name in names:
        assert append(lib, e4m3, **{name: N}) == -1, name
    for bad in (dict(rows=0), dict(rows=3), dict(seqs=0), dict(seqs=65536, rows=65536), dict(kvh=0), dict(dim=0),
                dict(dim=12, pairs=0), dict(dim=272), dict(pairs=33), dict(pairs=-1), dict(cols=0), dict(pages=0),
                dict(page=0), dict(code=2), dict(cols=1 << 20, page=1 << 12), dict(cols=(1 << 31) - 1023, page=1),
                dict(heads=-1), dict(heads=65536), dict(kc=ODD), dict(q=ODD), dict(q_out=ODD), dict(wq=ODD), dict(wk=ODD),
                dict(cache=(2048, 128, 4)), dict(cache=(-16, 128, 64)), dict(pages=1 << 30, cache=(1 << 11, 128, 64)),
                dict(strides=(256, 64, 128, 64, 130, 64)), dict(strides=(256, -64, 128, 64, 128, 64)), dict(eps=-1.0),
                dict(eps=float("nan"))):
        assert append(lib, e4m3, **bad) == -2, bad
        assert _lib.last_error()
    if e4m3:
        for bad in (dict(dim=8, pairs=4), dict(dim=72), dict(cache=(2048, 136, 64)), dict(scale=(-1, 16)), dict(scale=(32, -1)),
                    dict(scale=(1 << 41, 16))):
            assert append(lib, True, **bad) == -2, bad


def chunk(lib, e4m3, q=A, kc=A, vc=A, ks=A, vs=A, table=A, lengths=A, starts=A, out=A, scratch=N, nbytes=0, rows=2, seqs=2,
          heads=4, kvh=2, dim=64, strides=(256, 64), cols=64, pages=8, page=16, cache=(2048, 128, 64), scale=(32, 16), sm=0.125,
          code=1):
    if e4m3:
        return lib.kv_paged_attention_chunk_e4m3(q, kc, vc, ks, vs, table, lengths, starts, out, scratch, nbytes, rows, seqs,
                                                 heads, kvh, dim, *strides, cols, pages, page, *cache, *scale, sm, code)
    return lib.kv_paged_attention_chunk_u16(q, kc, vc, table, lengths, starts, out, scratch, nbytes, rows, seqs, heads, kvh,
                                            dim, *strides, cols, pages, page, *cache, sm, code)


@pytest.mark.parametrize("e4m3", [False, True])
def test_chunk_codes(lib, e4m3):
    for name in ["q", "kc", "vc", "table", "lengths", "starts", "out"] + (["ks", "vs"] if e4m3 else []):
        assert chunk(lib, e4m3, **{name: N}) == -1, name
    for bad in (dict(rows=0), dict(rows=1 << 30), dict(heads=3), dict(heads=0), dict(heads=1 << 17), dict(kvh=0), dict(seqs=0),
                dict(seqs=1 << 17), dict(dim=20), dict(dim=512), dict(code=2), dict(q=ODD), dict(out=ODD), dict(vc=ODD),
                dict(strides=(256, 63)), dict(strides=(-256, 64)), dict(cache=(2048, 127, 64)), dict(cols=1 << 28),
                dict(cols=1 << 21, page=1 << 10)):
        assert chunk(lib, e4m3, **bad) == -2, bad
        assert _lib.last_error()
    need = lib.kv_paged_attention_chunk_scratch_bytes(2, 2, 4, 2, 64, 64 * 16)
    assert need > 0
    assert chunk(lib, e4m3, scratch=A, nbytes=need - 1) == -3
    assert chunk(lib, e4m3, scratch=ODD, nbytes=need) == -3


def test_chunk_scratch(lib):
    need = lib.kv_paged_attention_chunk_scratch_bytes
    for bad in ((0, 2, 4, 2, 64, 64), (65536, 2, 4, 2, 64, 64), (2, 0, 4, 2, 64, 64), (2, 2, 3, 2, 64, 64), (2, 2, 4, 2, 0, 64),
                (2, 2, 4, 2, 264, 64), (2, 2, 4, 2, 64, 0), (2, 2, 4, 2, 64, 2 ** 31 - 1023), (2, 1 << 30, 4, 2, 64, 64)):
        assert need(*bad) == -2, bad
    assert need(1, 1, 4, 2, 64, 2 ** 31 - 1024) > 0
    assert need(1, 16384, 28, 4, 128, 16384) == 0  # tiles enough for the device
    # bounded, whatever the rows, sequences and positions
    for sequences in (1, 16, 256, 1000):
        for rows in (1, 37, 500, 5000):
            for heads, kvh, dim in ((28, 4, 128), (128, 128, 128), (32, 1, 64), (16, 4, 256)):
                assert 0 <= need(sequences, rows, heads, kvh, dim, 1 << 20) < 1 << 29


def decode(lib, q=A, kc=A, vc=A, ks=A, vs=A, table=A, lengths=A, out=A, scratch=N, nbytes=0, seqs=2, rows=1, heads=4, kvh=2,
           dim=64, strides=(256, 256, 64), cols=64, pages=8, page=16, cache=(2048, 128, 64), scale=(32, 16), sm=0.125, code=1):
    return lib.kv_paged_attention_decode_e4m3(q, kc, vc, ks, vs, table, lengths, out, scratch, nbytes, seqs, rows, heads, kvh,
                                              dim, *strides, cols, pages, page, *cache, *scale, sm, code)


def test_decode_codes(lib):
    for name in ("q", "kc", "vc", "ks", "vs", "table", "lengths", "out"):
        assert decode(lib, **{name: N}) == -1, name
    for bad in (dict(rows=0), dict(rows=9), dict(heads=3), dict(heads=0), dict(kvh=0), dict(seqs=0), dict(seqs=1 << 17),
                dict(dim=24), dict(dim=512), dict(code=2), dict(q=ODD), dict(out=ODD), dict(vc=ODD),
                dict(strides=(256, 256, 63)), dict(cache=(2048, 120, 64)), dict(cols=1 << 28), dict(scale=(-1, 16))):
        assert decode(lib, **bad) == -2, bad
    need = lib.kv_paged_attention_scratch_bytes(2, 1, 4, 2, 64, 64 * 16)
    assert decode(lib, scratch=A, nbytes=need - 1) == -3
    assert decode(lib, scratch=ODD, nbytes=need) == -3


@pytest.fixture
def no_device(monkeypatch):
    """The Python calls up to their first use of the device."""
    monkeypatch.setattr(native, "_require", lambda *a: None)


F16 = torch.float16
CACHE = torch.zeros((4, 16, 2, 64), dtype=F16)
CACHE8 = torch.zeros((4, 16, 2, 64), dtype=torch.uint8)
SCALES = torch.zeros((4, 2, 16))
Q, K, W = torch.zeros((3, 4, 64), dtype=F16), torch.zeros((3, 2, 64), dtype=F16), torch.zeros(64, dtype=F16)
TABLE, LENGTHS, STARTS = torch.zeros((3, 2), dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)


def norm_append(q=Q, k=K, v=K, wq=W, wk=W, kc=CACHE, vc=CACHE, table=TABLE, lengths=LENGTHS, rms_eps=1e-6, **kw):
    return native.kv_paged_norm_append(q, k, v, wq, wk, kc, vc, table, lengths, rms_eps=rms_eps, **kw)


def append8(q=Q, k=K, v=K, wq=None, wk=None, kc=CACHE8, vc=CACHE8, ks=SCALES, vs=SCALES, table=TABLE, lengths=LENGTHS, **kw):
    return native.kv_paged_append_e4m3(q, k, v, kc, vc, ks, vs, table, lengths, q_norm_weight=wq, k_norm_weight=wk, **kw)


def chunk16(q=Q, kc=CACHE, vc=CACHE, table=TABLE, lengths=LENGTHS, starts=STARTS):
    return native.kv_paged_attention_chunk(q, kc, vc, table, lengths, starts)


def chunk8(q=Q, kc=CACHE8, vc=CACHE8, ks=SCALES, vs=SCALES, table=TABLE, lengths=LENGTHS, starts=STARTS):
    return native.kv_paged_attention_chunk_e4m3(q, kc, vc, ks, vs, table, lengths, starts)


def decode8(q=Q, kc=CACHE8, vc=CACHE8, ks=SCALES, vs=SCALES, table=TABLE, lengths=LENGTHS):
    return native.kv_paged_attention_decode_e4m3(q, kc, vc, ks, vs, table, lengths)


@pytest.mark.parametrize("fn", [norm_append, append8, chunk16, chunk8, decode8])
def test_python_cache_refusals(no_device, fn):
    cases = [(dict(table=TABLE.long()), TypeError, "int32"), (dict(lengths=LENGTHS.long()), TypeError, "int32"),
             (dict(lengths=LENGTHS[:2]), ValueError, "one entry per sequence"),
             (dict(table=TABLE.repeat(1, 2)[:, ::2]), ValueError, "contiguous"), ({}, ValueError, "HIP device")]
    cache = CACHE if fn in (norm_append, chunk16) else CACHE8
    cases += [(dict(kc=cache.float(), vc=cache.float()), TypeError, "caches"), (dict(vc=cache[:2]), ValueError, "same strides"),
              (dict(kc=cache[0], vc=cache[0]), ValueError, "page_size"), (dict(vc=cache.to(torch.bfloat16)), TypeError, "caches")]
    if fn in (append8, chunk8, decode8):
        cases += [(dict(ks=SCALES.half()), TypeError, "float32"), (dict(vs=SCALES[:2]), ValueError, "scales must"),
                  (dict(ks=SCALES.transpose(1, 2), vs=SCALES.transpose(1, 2)), ValueError, "scales must"),
                  (dict(ks=SCALES.repeat(1, 1, 2)[..., ::2], vs=SCALES.repeat(1, 1, 2)[..., ::2]), ValueError, "adjacent slots"),
                  (dict(vs=SCALES.transpose(0, 1).contiguous().transpose(0, 1)), ValueError, "same strides")]
    for kw, err, text in cases:
        with pytest.raises(err, match=text):
            fn(**kw)


@pytest.mark.parametrize("fn", [norm_append, append8])
def test_python_append_refusals(no_device, fn):
    freq = torch.ones(32, dtype=torch.float64)
    for kw, err, text in ((dict(k=K.float()), TypeError, "rows"), (dict(v=K.bfloat16()), TypeError, "rows"),
                          (dict(v=K[:2]), ValueError, "kv_heads"), (dict(k=K[:, :1], v=K[:, :1]), ValueError, "kv_heads"),
                          (dict(q=Q[:2]), ValueError, "q must"), (dict(q=Q[:2], k=K[:2], v=K[:2]), ValueError, "multiple of the"),
                          (dict(row_starts=torch.zeros(4)), TypeError, "row_starts"),
                          (dict(row_starts=STARTS[:3]), ValueError, "sequences \\+ 1"),
                          (dict(rope_frequencies=freq.float()), TypeError, "float64"),
                          (dict(rope_frequencies=freq.repeat(2)), ValueError, "head_dim / 2"),
                          (dict(rejected=torch.zeros(1)), TypeError, "rejected"), (dict(rms_eps=-1.0), ValueError, "negative"),
                          (dict(rms_eps=float("nan")), ValueError, "negative")):
        with pytest.raises(err, match=text):
            fn(**kw)
    if fn is norm_append:
        for kw in (dict(wq=None), dict(wk=None)):
            with pytest.raises(TypeError, match="norm weights"):
                fn(**kw)


def test_python_norm_weight_refusals(no_device, monkeypatch):
    monkeypatch.setattr(native, "_on_device", lambda *a: 0)
    for fn in (norm_append, append8):
        for kw, err in ((dict(wq=W.bfloat16(), wk=W), TypeError), (dict(wq=W, wk=W.float()), TypeError),
                        (dict(wq=W[:32], wk=W), ValueError), (dict(wq=W, wk=W[None]), ValueError)):
            with pytest.raises(err, match="norm weights"):
                fn(**kw)


@pytest.mark.parametrize("fn", [chunk16, chunk8])
def test_python_chunk_refusals(no_device, fn):
    for kw, err, text in ((dict(q=Q[0]), ValueError, "q must"), (dict(q=Q[..., :32]), ValueError, "q must"),
                          (dict(q=Q[:, :3]), ValueError, "multiple of kv_heads"), (dict(q=Q[:, :0]), ValueError, "multiple of kv"),
                          (dict(q=Q.float()), TypeError, "requires"), (dict(starts=STARTS.long()), TypeError, "row_starts"),
                          (dict(starts=STARTS[:3]), ValueError, "sequences \\+ 1"),
                          (dict(starts=torch.zeros(8, dtype=torch.int32)[::2]), ValueError, "sequences \\+ 1")):
        with pytest.raises(err, match=text):
            fn(**kw)


def test_python_decode_refusals(no_device):
    for kw, text in ((dict(q=Q[:, :3]), "multiple of kv_heads"), (dict(q=Q[:2]), "q must"), (dict(q=Q[:, 0]), "q must"),
                     (dict(q=Q[:, None].expand(3, 9, 4, 64)), "1 to 8 rows"), (dict(q=Q[:, None][:, :0]), "1 to 8 rows")):
        with pytest.raises(ValueError, match=text):
            decode8(**kw)


def test_kill_switch(monkeypatch):
    monkeypatch.setenv("PCKETLM_DISABLE_NATIVE_KV", "1")
    for fn in (norm_append, append8, chunk16, chunk8, decode8):
        with pytest.raises(RuntimeError, match="unavailable: disabled"):
            fn()
