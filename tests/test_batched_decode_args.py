"""What the batched decode operators refuse, on the CPU: the C entry points'
codes (no check reaches a device), and the exceptions of the Python calls."""

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


def test_rows_codes(lib):
    assert lib.fp8_e4m3_quantize_rows(N, A, A, 1, 8, 8, 1) == -1
    for rows, cols, stride, code in ((0, 8, 8, 1), (1, 0, 8, 1), (1, 65537, 8, 1), (1, 8, -8, 1), (1, 8, 8, 3),
                                     (1, 8, 8, -1)):
        assert lib.fp8_e4m3_quantize_rows(A, A, A, rows, cols, stride, code) == -2
    assert lib.fp8_e4m3_rms_norm_rows(A, N, N, N, A, A, 1, 8, 8, 0, 1, 1e-6) == -1   # no weight
    assert lib.fp8_e4m3_rms_norm_rows(A, A, A, N, A, A, 1, 8, 8, 8, 1, 1e-6) == -1   # a residual, no sum
    assert lib.fp8_e4m3_rms_norm_rows(A, A, A, A, A, A, 1, 8, 8, -1, 1, 1e-6) == -2
    assert lib.fp8_e4m3_rms_norm_rows(A, N, A, N, A, A, 1, 1 << 20, 8, 0, 0, 1e-6) == -2


def test_matmul_codes(lib):
    def call(x=A, xs=A, w=A, ws=A, out=A, scratch=N, nbytes=0, m=1, n=16, k=128, sc=1, code=1):
        return lib.fp8_e4m3_block_matmul(x, xs, w, ws, out, scratch, nbytes, m, n, k, sc, code)

    for name in ("x", "xs", "w", "ws", "out"):
        assert call(**{name: N}) == -1
    for bad in (dict(m=0), dict(n=-1), dict(k=0), dict(k=129), dict(code=3), dict(m=1 << 31), dict(n=1 << 31), dict(x=ODD), dict(w=ODD)):
        assert call(**bad) == -2
    assert lib.fp8_e4m3_block_matmul_scratch_bytes(0, 1, 1, 1) == -2
    assert lib.fp8_e4m3_block_matmul_scratch_bytes(1, 1, 1, 3) == -2
    need = lib.fp8_e4m3_block_matmul_scratch_bytes(64, 7168, 16384, 1)
    assert need > 0
    assert call(m=64, n=7168, k=16384, sc=128, scratch=A, nbytes=need - 1) == -3
    assert call(m=64, n=7168, k=16384, sc=128, scratch=ODD, nbytes=need) == -3


def append(lib, q=A, k=A, v=A, q_out=A, kc=A, vc=A, table=A, lengths=A, starts=N, freq=A, rejected=N, rows=2, seqs=2,
           heads=4, kvh=2, dim=64, pairs=32, inter=0, strides=(256, 64, 128, 64, 128, 64), cols=4, pages=8, page=16,
           cache=(2048, 128, 64), code=1):
    return lib.kv_paged_append_u16(q, k, v, q_out, kc, vc, table, lengths, starts, freq, rejected, rows, seqs, heads, kvh,
                                   dim, pairs, inter, *strides, cols, pages, page, *cache, code)


def test_append_codes(lib):
    for name in ("q", "k", "v", "q_out", "kc", "vc", "table", "lengths", "freq"):
        assert append(lib, **{name: N}) == -1, name
    for bad in (dict(rows=0), dict(rows=3), dict(seqs=0), dict(seqs=65536, rows=65536), dict(kvh=0), dict(dim=0),
                dict(dim=12, pairs=0), dict(dim=264), dict(pairs=33), dict(pairs=-1), dict(cols=0), dict(pages=0),
                dict(page=0), dict(code=2), dict(cols=1 << 20, page=1 << 12), dict(cols=1 << 21, page=1 << 10),
                dict(cols=(1 << 31) - 1023, page=1), dict(heads=-1), dict(kc=ODD), dict(q=ODD),
                dict(cache=(2048, 128, 4)), dict(cache=(-8, 128, 64)), dict(pages=1 << 30, cache=(1 << 10, 128, 64)),
                dict(strides=(256, 64, 128, 64, 130, 64)), dict(strides=(256, -64, 128, 64, 128, 64))):
        assert append(lib, **bad) == -2, bad
        assert _lib.last_error()


def attention(lib, q=A, kc=A, vc=A, table=A, lengths=A, out=A, scratch=N, nbytes=0, seqs=2, rows=1, heads=4, kvh=2, dim=64,
              strides=(256, 256, 64), cols=64, pages=8, page=16, cache=(2048, 128, 64), scale=0.125, code=1):
    return lib.kv_paged_attention_decode_u16(q, kc, vc, table, lengths, out, scratch, nbytes, seqs, rows, heads, kvh, dim,
                                             *strides, cols, pages, page, *cache, scale, code)


def test_attention_codes(lib):
    for name in ("q", "kc", "vc", "table", "lengths", "out"):
        assert attention(lib, **{name: N}) == -1, name
    for bad in (dict(rows=0), dict(rows=9), dict(heads=3), dict(heads=0), dict(kvh=0), dict(seqs=0), dict(seqs=1 << 17),
                dict(dim=20), dict(dim=512), dict(code=2), dict(q=ODD), dict(out=ODD), dict(vc=ODD),
                dict(strides=(256, 256, 63)), dict(cache=(2048, 127, 64)), dict(cols=1 << 28)):
        assert attention(lib, **bad) == -2, bad
    need = lib.kv_paged_attention_scratch_bytes(2, 1, 4, 2, 64, 64 * 16)
    assert need > 0
    assert attention(lib, scratch=A, nbytes=need - 1) == -3
    assert attention(lib, scratch=ODD, nbytes=need) == -3
    assert lib.kv_paged_attention_scratch_bytes(2, 1, 4, 2, 64, 512) == 0  # a workgroup for each sequence
    assert lib.kv_paged_attention_scratch_bytes(2, 1, 4, 2, 64, 513) > 0
    assert lib.kv_paged_attention_scratch_bytes(2, 9, 4, 2, 64, 128) == -2
    assert lib.kv_paged_attention_scratch_bytes(2, 1, 4, 2, 64, 0) == -2
    # positions are ints with room for two units behind the last
    assert lib.kv_paged_attention_scratch_bytes(1, 1, 4, 2, 64, 2 ** 31 - 1024) > 0
    assert lib.kv_paged_attention_scratch_bytes(1, 1, 4, 2, 64, 2 ** 31 - 1023) == -2
    assert attention(lib, cols=1 << 21, page=1 << 10) == -2


@pytest.fixture
def no_device(monkeypatch):
    """The Python calls up to their first use of the device."""
    monkeypatch.setattr(native, "_require", lambda *a: None)


def test_python_rows_refusals(no_device):
    x, w = torch.zeros((2, 256)), torch.zeros(256)
    with pytest.raises(TypeError, match="float32 rows"):
        native.fp8_e4m3_quantize_rows(x.double())
    with pytest.raises(ValueError, match="cols"):
        native.fp8_e4m3_quantize_rows(x[:, :0])
    with pytest.raises(ValueError, match="HIP device"):
        native.fp8_e4m3_quantize_rows(x)
    with pytest.raises(TypeError, match="share dtype"):
        native.fp8_e4m3_rms_norm_rows(x, w.half(), rms_eps=1e-6)
    with pytest.raises(TypeError, match="share dtype"):
        native.fp8_e4m3_rms_norm_rows(x, w, rms_eps=1e-6, residual=x.half())
    with pytest.raises(ValueError, match="per column"):
        native.fp8_e4m3_rms_norm_rows(x, w[:128], rms_eps=1e-6)
    with pytest.raises(ValueError, match="shape of x"):
        native.fp8_e4m3_rms_norm_rows(x, w, rms_eps=1e-6, residual=x[:1])
    with pytest.raises(ValueError, match="HIP device"):
        native.fp8_e4m3_rms_norm_rows(x, w, rms_eps=1e-6)


def test_python_matmul_refusals(no_device):
    rows = native.Fp8Rows(torch.zeros((3, 256), dtype=torch.uint8), torch.zeros((3, 2)))
    w, ws = torch.zeros((130, 256), dtype=torch.uint8), torch.zeros((2, 2))
    for args, kw, err, text in (
            ((rows, w, ws), dict(out_dtype=torch.float64), TypeError, "out_dtype"),
            ((native.Fp8Rows(rows.data.float(), rows.scales), w, ws), {}, TypeError, "e4m3"),
            ((rows, w.int(), ws), {}, TypeError, "e4m3"),
            ((rows, w, ws.half()), {}, TypeError, "float32"),
            ((native.Fp8Rows(rows.data[0], rows.scales), w, ws), {}, ValueError, "rows, in_cols"),
            ((rows, w[0], ws), {}, ValueError, "out_rows, in_cols"),
            ((rows, w[:, :128], ws), {}, ValueError, "do not match"),
            ((native.Fp8Rows(rows.data, rows.scales[:, :1]), w, ws), {}, ValueError, "each 128 columns"),
            ((rows, w, ws[:1]), {}, ValueError, "128x128 block layout"),
            ((rows, w, ws), {}, ValueError, "HIP device")):
        with pytest.raises(err, match=text):
            native.fp8_e4m3_block_matmul(*args, **kw)


def test_python_paged_refusals(no_device):
    cache = torch.zeros((4, 16, 2, 64), dtype=torch.float16)
    k = torch.zeros((3, 2, 64), dtype=torch.float16)
    q = torch.zeros((3, 4, 64), dtype=torch.float16)
    table, lengths = torch.zeros((3, 2), dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    freq = torch.ones(32, dtype=torch.float64)

    def append(q=q, k=k, v=k, kc=cache, vc=cache, table=table, lengths=lengths, **kw):
        return native.kv_paged_append(q, k, v, kc, vc, table, lengths, **kw)

    def attend(q=q, kc=cache, vc=cache, table=table, lengths=lengths, **kw):
        return native.kv_paged_attention_decode(q, kc, vc, table, lengths, **kw)

    for fn in (append, attend):
        for kw, err, text in ((dict(kc=cache.float(), vc=cache.float()), TypeError, "caches"),
                              (dict(vc=cache.bfloat16()), TypeError, "share dtype"),
                              (dict(q=q.bfloat16()), TypeError, "requires"),
                              (dict(table=table.long()), TypeError, "int32"),
                              (dict(lengths=lengths.long()), TypeError, "int32"),
                              (dict(vc=cache[:2]), ValueError, "same strides"),
                              (dict(vc=cache.transpose(0, 1).contiguous().transpose(0, 1)), ValueError, "same strides"),
                              (dict(kc=cache[0], vc=cache[0]), ValueError, "page_size"),
                              (dict(lengths=lengths[:2]), ValueError, "one entry per sequence"),
                              (dict(table=table.repeat(1, 2)[:, ::2]), ValueError, "contiguous"),
                              ({}, ValueError, "HIP device")):
            with pytest.raises(err, match=text):
                fn(**kw)
    for kw, err, text in ((dict(k=k.float()), TypeError, "rows"), (dict(v=k[:2]), ValueError, "kv_heads"),
                          (dict(k=k[:, :1], v=k[:, :1]), ValueError, "kv_heads"), (dict(q=q[:2]), ValueError, "q must"),
                          (dict(q=q[:2], k=k[:2], v=k[:2]), ValueError, "multiple of the sequences"),
                          (dict(row_starts=torch.zeros(4)), TypeError, "row_starts"),
                          (dict(row_starts=torch.zeros(3, dtype=torch.int32)), ValueError, "sequences \\+ 1"),
                          (dict(rope_frequencies=freq.float()), TypeError, "float64"),
                          (dict(rope_frequencies=freq.repeat(2)), ValueError, "head_dim / 2"),
                          (dict(rejected=torch.zeros(1)), TypeError, "rejected")):
        with pytest.raises(err, match=text):
            append(**kw)
    for kw, text in ((dict(q=q[:, :3]), "multiple of kv_heads"), (dict(q=q[:2]), "q must"), (dict(q=q[:, 0]), "q must"),
                     (dict(q=q[:, None].expand(3, 9, 4, 64)), "1 to 8 rows"), (dict(q=q[:, None][:, :0]), "1 to 8 rows")):
        with pytest.raises(ValueError, match=text):
            attend(**kw)


def test_kill_switches(monkeypatch):
    monkeypatch.setenv("PCKETLM_DISABLE_NATIVE_FP8_LINEAR", "1")
    monkeypatch.setenv("PCKETLM_DISABLE_NATIVE_KV", "1")
    assert native.native_fp8_rows_available() is False and native.native_paged_kv_available() is False
    x = torch.zeros((1, 128))
    with pytest.raises(RuntimeError, match="unavailable: disabled"):
        native.fp8_e4m3_quantize_rows(x)
    with pytest.raises(RuntimeError, match="unavailable: disabled"):
        native.kv_paged_append(None, x, x, x, x, x, x)


def test_attention_scratch_does_not_grow_with_the_sequences(lib):
    """A run leaves two partials at most, and there are as many runs for 512 sequences as for 65535: what
    grows is the deal's note of each sequence, 8 bytes."""
    need = lib.kv_paged_attention_scratch_bytes
    for rows, heads, kvh, dim, capacity in ((1, 64, 64, 128, 8192), (1, 128, 128, 128, 8192), (1, 32, 8, 128, 131072),
                                            (8, 28, 4, 128, 32768), (1, 16, 4, 256, 4096)):
        few = need(1000, rows, heads, kvh, dim, capacity)
        assert need(65535, rows, heads, kvh, dim, capacity) - few == 8 * (65535 - 1000)
        assert 0 < few < 1 << 28
