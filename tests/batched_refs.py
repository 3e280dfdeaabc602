"""The batched decode operators' definitions in 64 bits, on the CPU, and the
bounds that their rounding allows (see each function)."""

from __future__ import annotations

import math

import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}  # half the smallest step
U32 = 2.0 ** -24
E4M3_MAX = 448.0
SMALLEST_SCALE = 2.0 ** -126


def pad_blocks(t: torch.Tensor) -> torch.Tensor:
    cols = t.shape[-1]
    return torch.nn.functional.pad(t, (0, -cols % 128)).unflatten(-1, (-1, 128))


def row_scales(y: torch.Tensor) -> torch.Tensor:
    return (pad_blocks(y).abs().amax(-1) / E4M3_MAX).clamp(min=SMALLEST_SCALE)


def widen_scales(scales: torch.Tensor, cols: int) -> torch.Tensor:
    return scales.repeat_interleave(128, dim=-1)[..., :cols]


def half_step_e4m3(v: torch.Tensor) -> torch.Tensor:
    """Half a step of e4m3 at |v|: 4 significant bits from 2^-6, steps of 2^-9 below."""
    return torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 4)


def rms_norm(summed: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    s = summed.double()
    return s / torch.sqrt(s.square().mean(-1, keepdim=True) + eps) * weight.double()


def matmul(x, xs, w, ws):
    """(product, sum of the products' magnitudes) in 64 bits."""
    k, n = x.shape[1], w.shape[0]
    xf = x.view(torch.float8_e4m3fn).double() * widen_scales(xs.double(), k)
    grid = widen_scales(ws.double().repeat_interleave(128, dim=0)[:n], k)
    wf = w.view(torch.float8_e4m3fn).double() * grid
    return xf @ wf.t(), xf.abs() @ wf.abs().t()


def matmul_bound(want, size, x, xs, w, ws, dtype):
    """A sum in fp32 of blocks of 128 products, each step off by at most a
    whole step (2^-23: matrix instructions cut off rather than round) of the
    magnitudes' sum: 128 in a block, the scale's two products, one for each
    block and each join.  For a 16-bit result seven of each eight products of
    adjacent columns are also off by up to 2^-13 of the largest one's power of
    two (at most the product of the eights' largest values).  Then the output's
    rounding."""
    k, n = x.shape[1], w.shape[0]
    off = (128 + 4 + (k + 127) // 128 + 32) * 2.0 ** -23 * size
    if dtype != torch.float32:
        def largest(t, scales):
            t = torch.nn.functional.pad(t.view(torch.float8_e4m3fn).double().abs(), (0, -k % 8))
            return t.unflatten(1, (-1, 8)).amax(2) * scales.double().repeat_interleave(16, dim=1)[:, :(k + 7) // 8]

        off = off + 7 * 2.0 ** -13 * (largest(x, xs) @ largest(w, ws.repeat_interleave(128, dim=0)[:n]).t())
    return off + HALF[dtype] * (want.abs() + off) + TINY[dtype]


def places(page_table, lengths, rows, row_starts=None):
    """(sequence, position) of each row, None for rows of none."""
    out = []
    for r in range(rows):
        if row_starts is None:
            b, i = divmod(r, rows // len(lengths))
        else:
            b = max((s for s in range(len(lengths)) if row_starts[s] <= r < row_starts[s + 1]), default=None)
            if b is None:
                out.append(None)
                continue
            i = r - row_starts[b]
        out.append(None if lengths[b] < 0 else (b, lengths[b] + i))
    return out


def rotate(x, pos, freq, interleaved):
    """Head values [heads, head_dim] rotated to position pos, and the bound:
    sine and cosine within 4 steps of 2^-24 (the angle is reduced in 64 bits,
    rounded once below pi, and the functions' own error), three roundings of
    the products and the sum."""
    x = x.double()
    if freq is None or freq.numel() == 0:
        return x, torch.zeros_like(x)
    n = freq.numel()
    angle = pos * freq
    c, s = angle.cos(), angle.sin()
    out, mag = x.clone(), torch.zeros_like(x)
    a, b = (x[:, 0:2 * n:2], x[:, 1:2 * n:2]) if interleaved else (x[:, :n], x[:, n:2 * n])
    ya, yb, m = a * c - b * s, b * c + a * s, a.abs() + b.abs()
    if interleaved:
        out[:, 0:2 * n:2], out[:, 1:2 * n:2], mag[:, 0:2 * n:2], mag[:, 1:2 * n:2] = ya, yb, m, m
    else:
        out[:, :n], out[:, n:2 * n], mag[:, :n], mag[:, n:2 * n] = ya, yb, m, m
    return out, 8 * U32 * mag


def attention(q, k_cache, v_cache, page_table, lengths, scale):
    """(result, bound) for q [sequences, rows, heads, head_dim], everything on
    the CPU.  The bound: scores off by (head_dim + 4) 2^-23 of their products'
    magnitudes, which moves a weight by that share; weights rounded to the
    cache's type (half a step each) before the product with the values; exp2
    and the sums in fp32 (2^-22 and a step of 2^-23 for each of the positions
    and joins); the output's rounding."""
    dtype = q.dtype
    n, rows, heads, dim = q.shape
    pages, page, kvh, _ = k_cache.shape
    group = heads // kvh
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros(q.shape, dtype=torch.float64)
    for b in range(n):
        length = int(lengths[b])
        if length < 0:
            continue
        for r in range(rows):
            seen = [p for p in range(min(length + r + 1, page_table.shape[1] * page))
                    if 0 <= int(page_table[b, p // page]) < pages]
            if not seen:
                continue
            at = torch.tensor(seen)
            pg, slot = page_table[b][at // page].long(), at % page
            for h in range(kvh):
                k, v = k_cache[pg, slot, h].double(), v_cache[pg, slot, h].double()
                qs = q[b, r, h * group:(h + 1) * group].double()
                score = qs @ k.t() * scale
                off = (qs.abs() @ k.abs().t()) * abs(scale) * (dim + 4) * 2.0 ** -23
                p = torch.softmax(score, dim=1)
                o = p @ v
                share = HALF[dtype] + 2 * off + 2.0 ** -20 + (len(seen) / 32 + 64) * 2.0 ** -23
                wide = (p * share) @ v.abs() + share.amax(1, keepdim=True) * (p @ v.abs())
                out[b, r, h * group:(h + 1) * group] = o
                bound[b, r, h * group:(h + 1) * group] = wide + HALF[dtype] * (o.abs() + wide) + TINY[dtype]
    return out, bound


def within(got, want, bound, what=""):
    got, want = got.detach().cpu().double(), want.cpu().double()
    bad = ~((got - want).abs() <= bound.cpu()) & ~(got.isnan() & want.isnan())
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} off, first at "
                                 f"{bad.nonzero()[0].tolist()}: {got[bad][0]} against {want[bad][0]} "
                                 f"+- {bound.expand(want.shape)[bad.cpu()][0]}")


def make_pages(lens, page, kvh, dim, dtype, seed, *, extra_cols=1, spare=2):
    """Caches whose pages are dealt at random to sequences of at most `lens`
    positions; every slot holds N(0, 1) values, unused table entries -7."""
    g = torch.Generator().manual_seed(seed)
    per = [max(0, math.ceil(x / page)) for x in lens]
    total = sum(per) + spare
    order = torch.randperm(total, generator=g).tolist()
    table = torch.full((len(lens), max(max(per), 1) + extra_cols), -7, dtype=torch.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    k = torch.randn((total, page, kvh, dim), generator=g).to(dtype)
    v = torch.randn((total, page, kvh, dim), generator=g).to(dtype)
    return k, v, table
