"""Rows in e4m3 with a scale for each 128 columns, from rows as they are and
from the RMS norm of rows, against the definition in 64 bits."""

from __future__ import annotations

import pytest
import torch

import batched_refs as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nat():
    from pocketlm_amd import native

    assert native.native_fp8_rows_available(), "libpocketlm_hip.so must load on the GPU box"
    return native


def randn(shape, dtype, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def check_rows(rows, y, off):
    """rows against y [rows, cols], whose values may be off by the share `off`."""
    data, scales = rows.data.cpu(), rows.scales.cpu()
    assert data.dtype == torch.float8_e4m3fn and scales.dtype == torch.float32
    want = ref.row_scales(y)
    ref.within(scales, want, (off + 2 * ref.U32) * want, "scales")
    s = ref.widen_scales(scales.double(), y.shape[1])
    v = y / s
    # half a step, and what the value and the product with 1 / scale are off
    slack = (off + 4 * ref.U32) * v.abs() + 2.0 ** -40
    ref.within(data.double(), v.clamp(-448, 448), ref.half_step_e4m3(v.abs() + slack) + slack, "bytes")


# the largest a sum of squares over cols columns is off (as a share): 64 + 6 + 16 steps of the
# thread's, the wave's and the workgroup's sums, halved by the root, then six roundings
NORM_OFF = (86 / 2 + 6) * ref.U32


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 7168), (3, 1), (2, 127), (5, 129), (7, 128), (4, 1000), (600, 136),
                                       (1030, 3584), (2, 8200), (1, 20008), (1100, 520), (1, 65536), (1040, 9001)])
def test_norm_and_quantize_against_the_definition(nat, dtype, rows, cols):
    x, r = randn((rows, cols), dtype, cols), randn((rows, cols), dtype, cols + 1, 2.0)
    w = randn((cols,), dtype, cols + 2)
    got, summed = nat.fp8_e4m3_rms_norm_rows(x.cuda(), w.cuda(), rms_eps=1e-6, residual=r.cuda())
    want_sum = (x.float() + r.float()).to(dtype)
    assert torch.equal(summed.cpu(), want_sum)
    check_rows(got, ref.rms_norm(want_sum, w, 1e-6), NORM_OFF)
    alone, same = nat.fp8_e4m3_rms_norm_rows(want_sum.cuda(), w.cuda(), rms_eps=1e-6)
    assert torch.equal(same.cpu(), want_sum)
    assert torch.equal(alone.data.view(torch.uint8), got.data.view(torch.uint8)) and torch.equal(alone.scales, got.scales)
    check_rows(nat.fp8_e4m3_quantize_rows(x.cuda()), x.double(), 0.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quotients_are_rounded_once(nat, dtype):
    """Bytes are those of the fp32 quotient by the scale (half a step of fp32, then of
    e4m3): with 16-bit values many quotients lie on a border between two bytes."""
    x = randn((400, 2048), dtype, 9)
    got = nat.fp8_e4m3_quantize_rows(x.cuda())
    scales = got.scales.cpu()
    assert torch.equal(scales, ref.pad_blocks(x.float()).abs().amax(-1) / 448)
    want = (x.double() / ref.widen_scales(scales.double(), 2048)).float().clamp(-448, 448)
    assert torch.equal(got.data.cpu().float(), want.to(torch.float8_e4m3fn).float())


def test_rows_do_not_depend_on_the_batch(nat):
    """A row's bytes are the same alone (one workgroup of many waves) and in a
    long prompt (few waves) up to the order of its sum of squares; without the
    norm they are the same bits."""
    x = randn((1500, 896), torch.bfloat16, 3).cuda()
    every = nat.fp8_e4m3_quantize_rows(x)
    one = nat.fp8_e4m3_quantize_rows(x[777:778])
    assert torch.equal(every.data[777:778].view(torch.uint8), one.data.view(torch.uint8))
    assert torch.equal(every.scales[777:778], one.scales)


def test_strided_rows_and_leading_dimensions(nat):
    wide = randn((33, 3 * 640), torch.bfloat16, 4).cuda()
    x = wide[:, 640:1280]
    w = randn((640,), torch.bfloat16, 5).cuda()
    got, summed = nat.fp8_e4m3_rms_norm_rows(x, w, rms_eps=1e-5, residual=wide[:, :640])
    want, want_sum = nat.fp8_e4m3_rms_norm_rows(x.contiguous(), w, rms_eps=1e-5, residual=wide[:, :640].contiguous())
    assert torch.equal(summed, want_sum) and torch.equal(got.scales, want.scales)
    assert torch.equal(got.data.view(torch.uint8), want.data.view(torch.uint8))
    # one value off 16 bytes, and columns that are not adjacent
    odd = randn((9 * 257 + 1,), torch.float16, 6).cuda()[1:].view(9, 257)
    check_rows(nat.fp8_e4m3_quantize_rows(odd), odd.cpu().double(), 0.0)
    turned = randn((300, 40), torch.float32, 7).cuda().t()
    check_rows(nat.fp8_e4m3_quantize_rows(turned), turned.cpu().double(), 0.0)
    cube = randn((3, 5, 256), torch.float16, 8).cuda()
    out, same = nat.fp8_e4m3_rms_norm_rows(cube, w[:256].half(), rms_eps=1e-6, residual=cube)
    assert out.data.shape == (15, 256) and out.scales.shape == (15, 2) and same.shape == cube.shape
    empty = nat.fp8_e4m3_quantize_rows(torch.empty((0, 300), device="cuda"))
    assert empty.data.shape == (0, 300) and empty.scales.shape == (0, 3)


def test_extreme_blocks(nat):
    x = torch.zeros((7, 384))
    x[1, :128] = 1e-42            # below the smallest scale
    x[2, 128:256] = 3e38
    x[3, 5] = float("inf")
    x[4, 300] = float("nan")
    x[5] = torch.linspace(-1, 1, 384)
    x[6, 0], x[6, 1] = 448.0, 447.9
    got = nat.fp8_e4m3_quantize_rows(x.cuda())
    data, scales = got.data.cpu().float(), got.scales.cpu()
    assert torch.equal(scales[0], torch.full((3,), 2.0 ** -126)) and not data[0].any()
    assert scales[1, 0] == 2.0 ** -126 and not data[1].any()
    assert scales[2, 1] == torch.tensor(3e38) / 448 and torch.equal(data[2, 128:256], torch.full((128,), 448.0))
    assert scales[3].isnan().tolist() == [True, False, False] and data[3, :128].isnan().all() and not data[3, 128:].any()
    assert scales[4].isnan().tolist() == [False, False, True] and data[4, 256:].isnan().all() and not data[4, :256].any()
    check_rows(type(got)(got.data[5:], got.scales[5:]), x[5:].double(), 0.0)
    # through the norm a row with a NaN is NaN throughout, its neighbours are not touched
    rows, _ = nat.fp8_e4m3_rms_norm_rows(x[4:6].cuda(), torch.ones(384, device="cuda"), rms_eps=1e-6)
    assert rows.scales[0].isnan().all() and rows.data[0].float().isnan().all()
    check_rows(type(rows)(rows.data[1:], rows.scales[1:]), ref.rms_norm(x[5:6], torch.ones(384), 1e-6), NORM_OFF)


def test_the_c_entry_adds_in_place(nat):
    """out_sum may be x or the residual."""
    from pocketlm_amd import _lib

    lib = _lib.load()
    for which in ("x", "residual"):
        x, r = randn((40, 512), torch.bfloat16, 11).cuda(), randn((40, 512), torch.bfloat16, 12).cuda()
        w = randn((512,), torch.bfloat16, 13).cuda()
        want, summed = nat.fp8_e4m3_rms_norm_rows(x, w, rms_eps=1e-6, residual=r)
        data = torch.empty((40, 512), dtype=torch.uint8, device="cuda")
        scales = torch.empty((40, 4), device="cuda")
        lib.pocketlm_set_stream(torch.cuda.current_stream().cuda_stream)
        to = x if which == "x" else r
        assert lib.fp8_e4m3_rms_norm_rows(x.data_ptr(), r.data_ptr(), w.data_ptr(), to.data_ptr(), data.data_ptr(),
                                          scales.data_ptr(), 40, 512, 512, 512, 1, 1e-6) == 0
        assert torch.equal(to, summed) and torch.equal(data, want.data.view(torch.uint8))
        assert torch.equal(scales, want.scales)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(5, 7168), (7, 129), (1030, 520), (1100, 100), (601, 1500), (2, 20008), (1, 65536)])
def test_norm_of_rows_whose_squares_leave_fp32(nat, dtype, rows, cols):
    """Finite rows from near the type's largest value down to 2^-120, in one
    batch: the sum of squares passes fp32 both ways, y does not."""
    x = randn((rows, cols), torch.float32, cols + 3)
    powers = torch.tensor([124.0, 0.0, 63.0, -120.0, 90.0, -66.0, 64.0])[torch.arange(rows) % 7]
    x = (x * torch.exp2(powers)[:, None]).to(dtype)
    if rows > 1:
        x[1, 3] = 2.0 ** 100  # one value beside ordinary ones
    w = randn((cols,), dtype, cols + 4)
    for eps in (0.0, 1e-6):
        got, _ = nat.fp8_e4m3_rms_norm_rows(x.cuda(), w.cuda(), rms_eps=eps)
        check_rows(got, ref.rms_norm(x, w, eps), NORM_OFF)


def test_norm_rows_do_not_depend_on_the_batch(nat):
    """A row's norm alone (one workgroup of many waves) and in a long prompt
    (few waves): the order of the sum of squares differs, the bounds hold for
    both and the scales agree within them."""
    x, w = randn((1500, 896), torch.bfloat16, 14), randn((896,), torch.bfloat16, 15)
    every, _ = nat.fp8_e4m3_rms_norm_rows(x.cuda(), w.cuda(), rms_eps=1e-6)
    one, _ = nat.fp8_e4m3_rms_norm_rows(x[777:778].cuda(), w.cuda(), rms_eps=1e-6)
    want = ref.rms_norm(x, w, 1e-6)
    check_rows(every, want, NORM_OFF)
    check_rows(one, want[777:778], NORM_OFF)
