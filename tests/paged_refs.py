"""Definitions in 64 bits of the operators over prompts and e4m3 pages (any
device), and the bounds that their rounding allows (see each function)."""

from __future__ import annotations

import math

import torch

import batched_refs as ref

U32 = ref.U32
E4M3_MAX = ref.E4M3_MAX


def head_norm(x, weight, eps):
    """Heads [..., head_dim] normed, and the bound: a sum of head_dim squares in
    fp32 (half its relative error reaches the root), the mean, the root, the
    quotient and two products."""
    x = x.double()
    if weight is None:
        return x, torch.zeros_like(x)
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
    return y, ((x.shape[-1] + 8) / 2 + 6) * U32 * y.abs()


def normed_rotated(x, weight, eps, pos, freq, interleaved):
    """Heads [heads, head_dim] normed and rotated to pos, and the bound before
    the last rounding: the rotation's own (batched_refs.rotate), and the norm's
    error of both values of a pair."""
    y, off = head_norm(x, weight, eps)
    z, turned = ref.rotate(y, pos, freq, interleaved)
    if freq is None or freq.numel() == 0:
        return z, off
    n = freq.numel()
    moved = off.clone()
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    moved[:, a] = moved[:, b] = off[:, a] + off[:, b]
    return z, turned + moved


def quantized(z, off):
    """(bytes' values, scales, their bounds) of heads [..., head_dim] known to
    `off`: the scale is the largest value's error and a rounding off, a value
    over the scale half a step of e4m3 at most, both operands' errors moved in
    front of it."""
    top = z.abs().amax(-1)
    scale = (top / E4M3_MAX).clamp(min=ref.SMALLEST_SCALE)
    scale_off = off.amax(-1) / E4M3_MAX + U32 * scale
    u = z / scale[..., None]
    moved = off / scale[..., None] + u.abs() * (scale_off / scale)[..., None] + 2 * U32 * u.abs()
    return u, scale, ref.half_step_e4m3(u.abs() + moved) * (1 + 1e-12) + moved, scale_off


def gathered(cache, scales, table_row, tokens):
    """(values [tokens, kv_heads, head_dim] in 64 bits, which are there); pages
    that are not there give zeros."""
    pages, page = cache.shape[:2]
    at = torch.arange(tokens, device=cache.device)
    pid = table_row.to(cache.device)[at // page].long()
    there = (pid >= 0) & (pid < pages)
    pid, slot = torch.where(there, pid, 0), at % page
    if scales is None:
        values = cache[pid, slot].double()
    else:
        raw = cache if cache.dtype == torch.uint8 else cache.view(torch.uint8)
        values = raw[pid, slot].contiguous().view(torch.float8_e4m3fn).double() * scales[pid, :, slot].double()[..., None]
    return torch.where(there[:, None, None], values, 0.0), there


def chunk(q, k_cache, v_cache, table, lengths, starts, scale, *, scales=(None, None), weight=None):
    """(result, bound) of rows q [rows, heads, head_dim] by row starts.  What a
    row does not see takes no part, whatever it holds.

    The bound: scores off by (head_dim + 8) 2^-23 of their products' magnitudes
    (times the scales), which moves a weight by that share, the maximum's own
    by as much; weights off by `weight` (half a step of the type they are
    rounded to); exp2 and the sums in fp32 (2^-20, and a step of 2^-23 for each
    of the positions and joins); in fp16 a weight is cut to steps of 2^-24 of
    2^-7 of a maximum that may be the row's times 2^-8; the output's rounding."""
    dtype, (rows, heads, dim) = q.dtype, q.shape
    pages, page, kvh, _ = k_cache.shape
    group = heads // kvh
    weight = ref.HALF[dtype] if weight is None else weight
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for b in range(len(lengths)):
        length, first, last = int(lengths[b]), int(starts[b]), int(starts[b + 1])
        n = last - first
        if length < 0 or n <= 0:
            continue
        tokens = min(length + n, table.shape[1] * page)
        k, there = gathered(k_cache, scales[0], table[b], tokens)
        v, _ = gathered(v_cache, scales[1], table[b], tokens)
        at = torch.arange(tokens, device=q.device)
        for r0 in range(0, n, 256):
            r1 = min(n, r0 + 256)
            sees = there[None, :] & (at[None, :] <= length + torch.arange(r0, r1, device=q.device)[:, None])
            for h in range(kvh):
                qs = q[first + r0:first + r1, h * group:(h + 1) * group].double().transpose(0, 1).contiguous()  # [group, n, dim]
                kh, vh = k[:, h].contiguous(), v[:, h].contiguous()
                score = torch.matmul(qs, kh.t().contiguous()) * scale
                off = torch.matmul(qs.abs(), kh.t().abs().contiguous()) * abs(scale) * (dim + 8) * 2.0 ** -23
                off = torch.where(sees & score.isfinite(), off, 0.0)
                score = torch.where(sees, score, -math.inf)
                top = score.amax(2, keepdim=True)
                p = torch.exp(score - top) * sees
                p = torch.where(sees, p, 0.0)  # a NaN of what is not seen
                total = p.sum(2, keepdim=True)
                p = p / total
                if bool(torch.isfinite(vh).all()):
                    o, size = torch.matmul(p, vh), torch.matmul(p, vh.abs())
                else:
                    o = torch.where(sees[None, :, :, None], p[..., None] * vh, 0.0).sum(2)
                    size = o.abs()
                share = weight + 2 * off + 2.0 ** -20 + (tokens / 32 + 64) * 2.0 ** -23
                spread = torch.matmul(p * share, torch.nan_to_num(vh.abs(), posinf=0.0)) + share.amax(2, keepdim=True) * size
                if dtype == torch.float16 and scales[0] is None:
                    spread = spread + 2.0 ** -24 / total * torch.matmul(sees.double().expand(group, -1, -1).contiguous(),
                                                                        torch.nan_to_num(vh.abs(), posinf=0.0))
                none = ~sees.any(1)[None, :, None]
                o, spread = torch.where(none, 0.0, o), torch.where(none, 0.0, spread)
                to = (slice(first + r0, first + r1), slice(h * group, (h + 1) * group))
                out[to] = o.transpose(0, 1)
                bound[to] = (spread + ref.HALF[dtype] * (o.abs() + spread) + ref.TINY[dtype]).transpose(0, 1)
    return out, bound


def agree(got, want, bound, what=""):
    """Within the bound, infinities and NaN in the same places."""
    got, want, bound = got.double(), want.to(got.device), bound.to(got.device)
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~(((got - want).abs() <= bound) & want.isfinite()) & ~same
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: "
                                 f"{got[bad][0]} against {want[bad][0]} +- {bound[bad][0]}")


def make_pages(lens, page, kvh, dim, dtype, seed, *, device="cuda", extra_cols=1, spare=2, dirt=None):
    """(caches, scales, table): pages dealt at random to sequences of at most
    `lens` positions, N(0, 1) values (e4m3: N(0, 120) with scales between 4e-3
    and 9e-3), unused table entries -7.  dirt: what the slots behind each
    sequence's last position and the spare pages hold instead."""
    g = torch.Generator().manual_seed(seed)
    per = [max(0, math.ceil(x / page)) for x in lens]
    total = sum(per) + spare
    order = torch.randperm(total, generator=g).tolist()
    table = torch.full((len(lens), max(max(per), 1) + extra_cols), -7, dtype=torch.int32)
    used = torch.zeros((total, page), dtype=torch.bool)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        for p in range(n):
            used[order[at + p], :max(0, min(page, lens[b] - p * page))] = True
        at += n
    shape = (total, page, kvh, dim)
    caches, scales = [], [None, None]
    if dtype == torch.float8_e4m3fn:
        scales = []
    for _ in range(2):
        x = torch.randn(shape, generator=g)
        if dtype == torch.float8_e4m3fn:
            x = (x * 120).clamp(-E4M3_MAX, E4M3_MAX).to(dtype).view(torch.uint8)
            s = torch.rand((total, kvh, page), generator=g) * 5e-3 + 4e-3
            if dirt is not None:
                x[~used] = 0x7F
                s.transpose(1, 2)[~used] = dirt
            scales.append(s.to(device))
            caches.append(x.to(device).view(dtype))
        else:
            x = x.to(dtype)
            if dirt is not None:
                x[~used] = dirt
            caches.append(x.to(device))
    return caches, scales, table
