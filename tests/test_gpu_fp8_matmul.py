"""FP8 rows times an FP8 block-scaled weight, against the sum in 64 bits."""

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


def make(m, n, k, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((m, k), generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    w = torch.randn((n, k), generator=g).to(torch.float8_e4m3fn)
    xs = torch.rand((m, (k + 127) // 128), generator=g) * 9e-3 + 1e-3
    ws = torch.rand(((n + 127) // 128, (k + 127) // 128), generator=g) * 0.9 + 0.1
    return x, xs, w, ws


def run(nat, x, xs, w, ws, dtype):
    return nat.fp8_e4m3_block_matmul(nat.Fp8Rows(x.cuda(), xs.cuda()), w.cuda(), ws.cuda(), out_dtype=dtype)


SHAPES = [(1, 576, 7168), (1, 1, 16), (2, 130, 128), (8, 100, 144), (16, 128, 256), (17, 33, 400), (31, 257, 1536),
          (33, 200, 384), (63, 640, 896), (64, 1024, 1040), (65, 96, 272), (100, 513, 2048), (128, 256, 512),
          (129, 384, 4096), (200, 1000, 640), (255, 48, 16384), (257, 300, 1552), (500, 700, 1280), (1, 5000, 128),
          (300, 129, 130), (7, 40, 1), (5, 3, 137),
          (20, 300, 4096), (64, 200, 8192), (12, 400, 16384)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_against_64_bits(nat, dtype, m, n, k):
    x, xs, w, ws = make(m, n, k, m + n + k)
    got = run(nat, x, xs, w, ws, dtype)
    assert got.dtype == dtype and got.shape == (m, n)
    want, size = ref.matmul(x, xs, w, ws)
    ref.within(got, want, ref.matmul_bound(want, size, x, xs, w, ws, dtype))


# on 256 compute units: tiles of 32, 64, 128 (one and two workgroups on a unit) and 256 rows (one and two rounds),
# each with a share of the blocks and all of them, over rows and columns that end within a tile and a block
@pytest.mark.parametrize("m,n,k", [(2122, 132, 928), (401, 130, 2272), (2870, 257, 928), (453, 131, 3120),
                                   (2793, 655, 912), (2808, 129, 2896), (515, 6541, 912), (159, 5430, 10640),
                                   (1305, 6313, 912), (130, 5474, 9136), (1947, 8779, 944), (77, 3000, 3001)])
def test_every_tile(nat, m, n, k):
    x, xs, w, ws = make(m, n, k, m)
    want, size = ref.matmul(x, xs, w, ws)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        ref.within(run(nat, x, xs, w, ws, dtype), want, ref.matmul_bound(want, size, x, xs, w, ws, dtype), str(dtype))


@pytest.mark.parametrize("m,n,k", [(600, 2304, 1024), (1025, 1100, 528), (2048, 512, 896)])
def test_prompts(nat, m, n, k):
    x, xs, w, ws = make(m, n, k, m)
    want, size = ref.matmul(x, xs, w, ws)
    ref.within(run(nat, x, xs, w, ws, torch.bfloat16), want, ref.matmul_bound(want, size, x, xs, w, ws, torch.bfloat16))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [12, 16, 30, 64])
@pytest.mark.parametrize("k", [16384, 16400])
def test_weights_larger_than_the_caches(nat, m, k, dtype):
    n = 4200
    x, xs, w, ws = make(m, n, k, m)
    got = run(nat, x, xs, w, ws, dtype)
    for rows, grid in ((slice(0, 128), ws[:1]), (slice(4096, n), ws[32:])):
        want, size = ref.matmul(x, xs, w[rows], grid)
        ref.within(got[:, rows], want, ref.matmul_bound(want, size, x, xs, w[rows], grid, dtype))


def test_whole_numbers_are_exact(nat):
    """Small whole numbers and scales that are powers of two: every sum is exact."""
    g = torch.Generator().manual_seed(9)
    for m, n, k in ((3, 50, 640), (40, 300, 2176), (300, 520, 1280)):
        x = torch.randint(-4, 5, (m, k), generator=g).float().to(torch.float8_e4m3fn)
        w = torch.randint(-4, 5, (n, k), generator=g).float().to(torch.float8_e4m3fn)
        xs = torch.exp2(torch.randint(-2, 3, (m, k // 128), generator=g).float())
        ws = torch.exp2(torch.randint(-2, 3, ((n + 127) // 128, k // 128), generator=g).float())
        want, _ = ref.matmul(x, xs, w, ws)
        assert torch.equal(run(nat, x, xs, w, ws, torch.float32).cpu().double(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m", [3, 20, 60, 120, 400])
def test_outliers_that_cancel(nat, m, dtype):
    """Columns of large values that cancel each other: fp32 results keep the
    small ones, 16-bit results what the matrix cores leave of them."""
    n, k = 260, 2048
    x, xs, w, ws = make(m, n, k, m)
    xf, wf = x.float() / 60, w.float()
    xf[:, 5::128], xf[:, 70::128] = 448.0, -448.0
    wf[:, 70::128] = wf[:, 5::128]
    x, w = xf.to(torch.float8_e4m3fn), wf.to(torch.float8_e4m3fn)
    want, size = ref.matmul(x, xs, w, ws)
    ref.within(run(nat, x, xs, w, ws, dtype), want, ref.matmul_bound(want, size, x, xs, w, ws, dtype))


@pytest.mark.parametrize("m", [1, 20, 50, 90, 300])
def test_nan_rows_weights_and_scales_stay_where_they_are(nat, m):
    n, k = 200, 656
    x, xs, w, ws = make(m, n, k, 21)
    want, size = ref.matmul(x, xs, w, ws)
    bound = ref.matmul_bound(want, size, x, xs, w, ws, torch.bfloat16)
    xb, wb, xs2 = x.view(torch.uint8).clone(), w.view(torch.uint8).clone(), xs.clone()
    wb[17, k - 1] = 0x7F
    wb[199, 0] = 0xFF
    if m > 1:
        xb[m - 1, 3] = 0x7F
        xs2[m // 2, 5] = float("nan")
    got = run(nat, xb, xs2, wb, ws, torch.bfloat16).cpu()
    hit = torch.zeros((m, n), dtype=torch.bool)
    hit[:, 17] = hit[:, 199] = True
    if m > 1:
        hit[m - 1] = hit[m // 2] = True
    assert torch.equal(got.isnan(), hit)
    ref.within(got[~hit], want[~hit], bound[~hit])


def test_offset_and_strided_operands(nat):
    m, n, k = 70, 150, 512
    x, xs, w, ws = make(m, n, k, 30)
    want = run(nat, x, xs, w, ws, torch.float32)
    wide = torch.zeros((m, 2 * k), dtype=torch.uint8, device="cuda")
    wide[:, k:] = x.cuda().view(torch.uint8)
    odd = torch.zeros(n * k + 1, dtype=torch.uint8, device="cuda")[1:].view(n, k)
    odd.copy_(w.cuda().view(torch.uint8))
    got = nat.fp8_e4m3_block_matmul(nat.Fp8Rows(wide[:, k:], xs.cuda()), w.cuda(), ws.cuda().t().contiguous().t(),
                                    out_dtype=torch.float32)
    assert torch.equal(got, want)
    exact, size = ref.matmul(x, xs, w, ws)
    # an odd address: copied first
    ref.within(nat.fp8_e4m3_block_matmul(nat.Fp8Rows(x.cuda(), xs.cuda()), odd, ws.cuda(), out_dtype=torch.float32),
               exact, ref.matmul_bound(exact, size, x, xs, w, ws, torch.float32))
    assert nat.fp8_e4m3_block_matmul(nat.Fp8Rows(x.cuda()[:0], xs.cuda()[:0]), w.cuda(), ws.cuda()).shape == (0, n)


def test_the_library_s_own_scratch(nat):
    """The C entry without scratch gives the bits of the call with it."""
    from pocketlm_amd import _lib

    lib = _lib.load()
    for m, n, k in ((1, 300, 7168), (40, 256, 4096), (300, 384, 8192)):
        x, xs, w, ws = (t.cuda() for t in make(m, n, k, 40 + m))
        want = nat.fp8_e4m3_block_matmul(nat.Fp8Rows(x, xs), w, ws)
        out = torch.zeros_like(want)
        lib.pocketlm_set_stream(torch.cuda.current_stream().cuda_stream)
        assert lib.fp8_e4m3_block_matmul(x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), out.data_ptr(), None,
                                         0, m, n, k, k // 128, 1) == 0
        assert torch.equal(out, want)


def test_more_rows_than_a_grid_s_second_dimension_holds(nat):
    """More than 65535 tiles of 128 rows (a long batch through a narrow weight)."""
    m, n, k = 65535 * 128 + 300, 8, 16
    x, xs, w, ws = make(251, n, k, 50)
    of = torch.arange(m, device="cuda") % 251
    got = nat.fp8_e4m3_block_matmul(nat.Fp8Rows(x.view(torch.uint8).cuda()[of], xs.cuda()[of]), w.cuda(), ws.cuda(),
                                    out_dtype=torch.float32)
    want, size = ref.matmul(x, xs, w, ws)
    bound = ref.matmul_bound(want, size, x, xs, w, ws, torch.float32)
    assert bool(((got.double() - want.cuda()[of]).abs() <= bound.cuda()[of]).all())


@pytest.mark.parametrize("m,n,k,dtype", [
    (18, 12967, 5936, torch.bfloat16), (91, 14964, 6800, torch.bfloat16), (128, 12332, 7728, torch.float16),
    (420, 4202, 16352, torch.float32), (64, 37888, 3584, torch.bfloat16), (40, 33000, 2048, torch.float32),
    (16, 33000, 2048, torch.bfloat16), (60, 24576, 4096, torch.bfloat16)])
def test_large_weights_and_groups_of_rows(nat, m, n, k, dtype):
    """Weights larger than the caches under one group of rows and several, in one share of the columns and several."""
    x, xs, w, ws = make(m, n, k, m)
    got = run(nat, x, xs, w, ws, dtype)
    last = (n - 1) // 128
    for rows, grid in ((slice(0, 256), ws[:2]), (slice(128 * (last // 2), 128 * (last // 2) + 128), ws[last // 2:last // 2 + 1]),
                       (slice(128 * last, n), ws[last:])):
        want, size = ref.matmul(x, xs, w[rows], grid)
        ref.within(got[:, rows], want, ref.matmul_bound(want, size, x, xs, w[rows], grid, dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(3, 50, 640), (12, 400, 16384), (40, 300, 2176), (64, 640, 16384), (300, 520, 1280),
                                   (515, 6541, 896), (1947, 8779, 944)])
def test_whole_numbers_are_exact_in_16_bits(nat, m, n, k, dtype):
    """Small whole numbers and scales that are powers of two: no product of at
    most 16 is cut off beside another, every sum is exact, and the result is
    rounded once."""
    g = torch.Generator().manual_seed(m)
    x = torch.randint(-4, 5, (m, k), generator=g).float().to(torch.float8_e4m3fn)
    w = torch.randint(-4, 5, (n, k), generator=g).float().to(torch.float8_e4m3fn)
    xs = torch.exp2(torch.randint(-2, 3, (m, (k + 127) // 128), generator=g).float())
    ws = torch.exp2(torch.randint(-2, 3, ((n + 127) // 128, (k + 127) // 128), generator=g).float())
    want, size = ref.matmul(x, xs, w, ws)
    # every partial sum is a multiple of 1/16 below 2^20: 24 bits hold it
    assert float(size.max()) < 2 ** 20
    assert torch.equal(run(nat, x, xs, w, ws, dtype).cpu(), want.to(dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [5, 17, 32, 33, 64, 200])
@pytest.mark.parametrize("n,k", [(32769, 1040), (70000, 256)])
def test_weights_of_more_tiles_than_compute_units(nat, m, n, k, dtype):
    """Fused projections and vocabularies: several rounds of weight tiles."""
    x, xs, w, ws = make(m, n, k, m)
    got = run(nat, x, xs, w, ws, dtype)
    assert got.shape == (m, n)
    for first in (0, 128 * (n // 384), n // 128 * 128):
        rows, grid = slice(first, min(first + 128, n)), ws[first // 128:first // 128 + 1]
        want, size = ref.matmul(x, xs, w[rows], grid)
        ref.within(got[:, rows], want, ref.matmul_bound(want, size, x, xs, w[rows], grid, dtype))


def test_only_the_operand_at_an_odd_address_is_copied(nat):
    m, n, k = 3, 4096, 2048
    x, xs, w, ws = (t.cuda() for t in make(m, n, k, 31))
    want = nat.fp8_e4m3_block_matmul(nat.Fp8Rows(x, xs), w, ws)
    odd = torch.zeros(m * k + 1, dtype=torch.uint8, device="cuda")[1:].view(m, k)
    odd.copy_(x.view(torch.uint8))
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got = nat.fp8_e4m3_block_matmul(nat.Fp8Rows(odd, xs), w, ws)
    assert torch.equal(got, want)
    assert torch.cuda.max_memory_allocated() - before < n * k  # the rows, the result and the scratch
