"""The operators of a batched decode step over FP8 weights and a paged cache, as cases to measure.

  norm       a residual's addition and the RMS norm of the sum, its rows in e4m3 with a scale for
             each 128 columns
  product    rows in e4m3 with such scales times an FP8 block-scaled weight (a scale for each
             128 x 128 block)
  append     rows of keys and values rotated to their positions and written into the pages of their
             sequences, the queries rotated along
  attention  one to eight new query rows of each sequence over its pages

`run` computes them either in their plain form (elementary torch operations in 32 bits, positions'
angles in 64) or, where `own` is true, through pocketlm_amd.native.  Sizes are those of the
repository's benchmark (DeepSeek-V3 shaped projections, a Qwen2.5-7B shaped dense layer) and generic
ones.  Weights are N(0, 0.02) cast to e4m3 with scales uniform in (1e-3, 1e-2), 16-bit values N(0, 1).
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3_MAX = 448.0
SMALLEST_SCALE = 2.0 ** -126


def listed():
    return [
        # the input norm of one generated token
        {"name": "norm_one_token", "kind": "norm", "rows": 1, "cols": 7168, "dtype": "bf16", "residual": True},
        # a prompt chunk of ragged length through a dense layer's norm
        {"name": "norm_chunk", "kind": "norm", "rows": 509, "cols": 3584, "dtype": "fp16", "residual": True},
        # a long prompt's rows
        {"name": "norm_prompt", "kind": "norm", "rows": 8192, "cols": 7168, "dtype": "bf16", "residual": True},
        # the smallest projection of one generated token
        {"name": "product_one_token", "kind": "product", "rows": 1, "out": 576, "cols": 7168, "dtype": "bf16"},
        # a batch of decoding sequences through the largest projection
        {"name": "product_batch", "kind": "product", "rows": 64, "out": 7168, "cols": 16384, "dtype": "bf16"},
        # a prompt chunk of ragged length through the query up-projection
        {"name": "product_chunk", "kind": "product", "rows": 509, "out": 24576, "cols": 1536, "dtype": "bf16"},
        # a long prompt through the largest projection
        {"name": "product_prompt", "kind": "product", "rows": 4096, "out": 7168, "cols": 16384, "dtype": "bf16"},
        # one step of a batch of decoding sequences
        {"name": "append_batch", "kind": "append", "sequences": 64, "rows": 1, "heads": 28, "kv_heads": 4, "head": 128,
         "page": 16, "context": 1000, "ragged": True, "dtype": "bf16"},
        # a few prompts of ragged lengths into an empty cache
        {"name": "append_prompts", "kind": "append", "sequences": 5, "rows": 1700, "heads": 28, "kv_heads": 4,
         "head": 128, "page": 64, "context": 0, "ragged": True, "dtype": "fp16"},
        # one sequence, a short conversation: the latency of the call
        {"name": "attention_short", "kind": "attention", "sequences": 1, "rows": 1, "heads": 28, "kv_heads": 4,
         "head": 128, "page": 16, "context": 700, "ragged": False, "dtype": "fp16"},
        # a speculative verifier's four rows of each of a few sequences of ragged lengths
        {"name": "attention_verifier", "kind": "attention", "sequences": 6, "rows": 4, "heads": 28, "kv_heads": 4,
         "head": 128, "page": 32, "context": 5003, "ragged": True, "dtype": "bf16"},
        # a server's batch of long conversations
        {"name": "attention_batch", "kind": "attention", "sequences": 48, "rows": 1, "heads": 28, "kv_heads": 4,
         "head": 128, "page": 16, "context": 16381, "ragged": True, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "product", "product", "append", "attention", "attention"])
    if kind == "norm":
        cols = _log(rng, 256, 7168)
        if rng.random() < 0.7:
            cols = max(256, cols // 128 * 128)
        return {"kind": kind, "rows": _log(rng, 1, 8192), "cols": cols,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "residual": rng.random() < 0.8}
    if kind == "product":
        cols = max(512, _log(rng, 512, 16384) // 16 * 16)
        out = _log(rng, 128, min(24576, 7168 * 16384 // cols))
        return {"kind": kind, "rows": _log(rng, 1, 4096), "out": out, "cols": cols,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    heads, kv_heads, head = rng.choice([(14, 2, 64), (12, 2, 128), (16, 8, 64), (32, 8, 64), (28, 4, 128), (16, 16, 64),
                                        (32, 1, 128), (8, 4, 256), (20, 5, 96)])
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "head": head,
            "page": rng.choice([8, 16, 16, 32, 64, 100, 128, 256]), "ragged": rng.random() < 0.7,
            "dtype": rng.choice(["fp16", "bf16"])}
    if kind == "append":
        if rng.random() < 0.5:
            return {**case, "sequences": _log(rng, 1, 64), "rows": rng.choice([1, 1, 2, 4, 8]),
                    "context": _log(rng, 16, 2000)}
        return {**case, "sequences": rng.randint(1, 5), "rows": _log(rng, 16, 1700), "context": rng.choice([0, 0, 333])}
    # at most the bytes of the largest listed cache
    context = _log(rng, 16, 32768)
    most = 48 * 16381 * 4 * 128 // (context * kv_heads * head)
    return {**case, "sequences": _log(rng, 1, max(1, min(64, most))), "rows": rng.choice([1, 1, 1, 2, 4, 8]),
            "context": context}


# ---------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(shape, g, dtype, std=1.0):
    """N(0, std) in `dtype`, made a piece at a time where it is large."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    step = 1 << 27
    for at in range(0, flat.numel(), step):
        n = min(step, flat.numel() - at)
        flat[at:at + n] = (torch.randn(n, generator=g, device="cuda") * std).to(dtype)
    return out


def _blocks(n):
    return (n + 127) // 128


def _spread(most, count, ragged):
    """`count` sizes, the largest `most`; ragged ones go down to about half of it."""
    return [max(0, int(round(most * (1.0 - 0.5 * i / count)))) if ragged else most for i in range(count)]


def _sizes(case):
    """The tokens that each sequence has before the call, and its new rows."""
    n = case["sequences"]
    if case["kind"] == "append" and case["rows"] > 8:
        return _spread(case["context"], n, False), [max(1, r) for r in _spread(case["rows"], n, case["ragged"])]
    before = [max(0, c - case["rows"]) for c in _spread(case["context"], n, case["ragged"])]
    return before, [case["rows"]] * n


def _cache(case, g, before, rows):
    """Caches with every page at a random place, and each sequence's pages."""
    page, kvh, head = case["page"], case["kv_heads"], case["head"]
    per = [(b + r + page - 1) // page for b, r in zip(before, rows)]
    total, widest = sum(per), max(per)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    per_t = torch.tensor(per, device="cuda")
    first = torch.cumsum(per_t, 0) - per_t
    at = torch.arange(widest, device="cuda")
    inside = at[None, :] < per_t[:, None]
    table = torch.where(inside, order[(first[:, None] + at[None, :]).clamp(max=total - 1)], torch.zeros_like(order[:1]))
    shape = (total, page, kvh, head)
    dtype = DTYPES[case["dtype"]]
    return {"k_cache": _randn(shape, g, dtype), "v_cache": _randn(shape, g, dtype),
            "page_table": table.to(torch.int32).contiguous(),
            "lengths": torch.tensor(before, dtype=torch.int32, device="cuda")}


def prepare(case, seed):
    g = _gen(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    state = {"case": case, "dtype": dtype}
    if kind == "norm":
        shape = (case["rows"], case["cols"])
        state["x"] = _randn(shape, g, dtype)
        state["residual"] = _randn(shape, g, dtype) if case["residual"] else None
        state["weight"] = (1.0 + 0.1 * torch.randn(case["cols"], generator=g, device="cuda")).to(dtype)
        return state
    if kind == "product":
        rows, out, cols = case["rows"], case["out"], case["cols"]
        nb = _blocks(cols)
        # activations as a quantizer leaves them: the largest of each 128 near e4m3's largest value
        state["x"] = (_randn((rows, cols), g, torch.float32) * 120.0).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        state["x_scales"] = torch.rand((rows, nb), generator=g, device="cuda") * 8e-3 + 4e-3
        state["w"] = _randn((out, cols), g, torch.float8_e4m3fn, 0.02)
        state["w_scales"] = torch.rand((_blocks(out), nb), generator=g, device="cuda") * 9e-3 + 1e-3
        return state
    before, rows = _sizes(case)
    heads, kvh, head = case["heads"], case["kv_heads"], case["head"]
    state.update(_cache(case, g, before, rows))
    if kind == "attention":
        q = _randn((case["sequences"], case["rows"], heads, head), g, dtype)
        state["q"] = q[:, 0] if case["rows"] == 1 else q
        return state
    # q, k and v as the fused projection leaves them: columns of one matrix
    total = sum(rows)
    qkv = _randn((total, (heads + 2 * kvh) * head), g, dtype)
    q, k, v = qkv.split([heads * head, kvh * head, kvh * head], dim=1)
    state["q"], state["k"], state["v"] = (t.unflatten(1, (-1, head)) for t in (q, k, v))
    state["frequencies"] = torch.tensor([1e6 ** (-2.0 * i / head) for i in range(head // 2)], dtype=torch.float64,
                                        device="cuda")
    state["row_starts"] = None
    if case["rows"] > 8:
        starts = [0]
        for r in rows:
            starts.append(starts[-1] + r)
        state["row_starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    return state


# ---------------------------------------------------------------- the plain forms

def _padded(t, cols):
    """The last dimension padded with zeros to whole blocks of 128."""
    return torch.nn.functional.pad(t, (0, _blocks(cols) * 128 - cols))


def _norm(s):
    x, cols, dtype = s["x"], s["case"]["cols"], s["dtype"]
    summed = x if s["residual"] is None else (x.float() + s["residual"].float()).to(dtype)
    h = summed.float()
    y = h * torch.rsqrt((h * h).mean(dim=1, keepdim=True) + 1e-6) * s["weight"].float()
    blocks = _padded(y, cols).unflatten(1, (-1, 128))
    scales = (blocks.abs().amax(dim=2) / E4M3_MAX).clamp(min=SMALLEST_SCALE)
    q = (blocks / scales[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).flatten(1)[:, :cols].to(torch.float8_e4m3fn)
    return {"rows": q, "scales": scales, "sum": summed}


def _product(s):
    rows, out, cols = s["case"]["rows"], s["case"]["out"], s["case"]["cols"]
    x = s["x"].float() * s["x_scales"].repeat_interleave(128, dim=1)[:, :cols]
    grid = s["w_scales"].repeat_interleave(128, dim=0)[:out].repeat_interleave(128, dim=1)[:, :cols]
    return torch.matmul(x, (s["w"].float() * grid).t()).to(s["dtype"])


def _row_places(s):
    """The sequence and the position of each new row."""
    lengths = s["lengths"].long()
    if s["row_starts"] is None:
        r = s["case"]["rows"]
        n = torch.arange(lengths.numel() * r, device="cuda")
        return n // r, lengths[n // r] + n % r
    starts = s["row_starts"].long()
    n = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(starts, n, right=True) - 1
    return seq, lengths[seq] + n - starts[seq]


def _rotate(x, cos, sin, dtype):
    a, b = x.float().chunk(2, dim=2)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=2).to(dtype)


def _append(s):
    seq, pos = _row_places(s)
    angle = pos.double()[:, None] * s["frequencies"][None, :]
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    page = s["case"]["page"]
    to = (s["page_table"][seq, pos // page].long(), pos % page)
    s["k_cache"][to] = _rotate(s["k"], cos, sin, s["dtype"])
    s["v_cache"][to] = s["v"]
    return {"q": _rotate(s["q"], cos, sin, s["dtype"]), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attention(s):
    case = s["case"]
    page, kvh, head, rows = case["page"], case["kv_heads"], case["head"], case["rows"]
    group, n = case["heads"] // kvh, case["sequences"]
    length = s["page_table"].shape[1] * page
    at = torch.arange(length, device="cuda")
    pages = s["page_table"].long()[:, at // page]
    k = s["k_cache"][pages, at % page].permute(0, 2, 3, 1).contiguous().float()  # [n, kvh, head, length]
    v = s["v_cache"][pages, at % page].permute(0, 2, 1, 3).contiguous().float()  # [n, kvh, length, head]
    q = s["q"].reshape(n, rows, kvh, group, head).permute(0, 2, 1, 3, 4).reshape(n, kvh, rows * group, head).float()
    seen = s["lengths"].long()[:, None] + 1 + torch.arange(rows, device="cuda")[None, :]
    hidden = at[None, None, :] >= seen[:, :, None]
    scores = torch.matmul(q, k) * (1.0 / math.sqrt(head))
    scores.masked_fill_(hidden[:, None, :, None, :].expand(n, 1, rows, group, length).reshape(n, 1, rows * group, length),
                        -math.inf)
    p = torch.exp(scores - scores.amax(dim=3, keepdim=True))
    out = torch.matmul(p, v) / p.sum(dim=3, keepdim=True)
    out = out.view(n, kvh, rows, group, head).permute(0, 2, 1, 3, 4).reshape(n, rows, kvh * group, head).to(s["dtype"])
    return out[:, 0] if rows == 1 else out


# ---------------------------------------------------------------- a pass

def _own(s):
    from pocketlm_amd import native

    kind = s["case"]["kind"]
    if kind == "norm":
        rows, summed = native.fp8_e4m3_rms_norm_rows(s["x"], s["weight"], rms_eps=1e-6, residual=s["residual"])
        return {"rows": rows.data, "scales": rows.scales, "sum": summed}
    if kind == "product":
        return native.fp8_e4m3_block_matmul(native.Fp8Rows(s["x"], s["x_scales"]), s["w"], s["w_scales"],
                                            out_dtype=s["dtype"])
    if kind == "append":
        q = native.kv_paged_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["page_table"], s["lengths"],
                                   row_starts=s["row_starts"], rope_frequencies=s["frequencies"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    return native.kv_paged_attention_decode(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["lengths"])


def run(state):
    if own:
        return _own(state)
    return {"norm": _norm, "product": _product, "append": _append, "attention": _attention}[state["case"]["kind"]](state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    kind = case["kind"]
    size = 4 if case["dtype"] == "fp32" else 2
    if kind == "norm":
        n = case["rows"] * case["cols"]
        moved = n * (size * (3 if case["residual"] else 1) + 1) + case["rows"] * _blocks(case["cols"]) * 4
        return {"bytes": moved + case["cols"] * size, "flops": 6 * n}
    if kind == "product":
        rows, out, cols = case["rows"], case["out"], case["cols"]
        return {"bytes": rows * cols + out * cols + 4 * _blocks(cols) * (rows + _blocks(out)) + rows * out * size,
                "flops": 2 * rows * out * cols}
    before, rows = _sizes(case)
    heads, kvh, head = case["heads"], case["kv_heads"], case["head"]
    if kind == "append":
        total = sum(rows)
        return {"bytes": 2 * total * (heads + 2 * kvh) * head * size, "flops": 3 * total * (heads + kvh) * head}
    seen = sum(b + r for b, r in zip(before, rows))
    new = sum(rows)
    pairs = sum(r * (b + (r + 1) / 2) for b, r in zip(before, rows))
    return {"bytes": 2 * seen * kvh * head * size + 2 * new * heads * head * size, "flops": 4 * pairs * heads * head}


# ---------------------------------------------------------------- the definition in 64 bits

def _exact_norm(s):
    cols = s["case"]["cols"]
    summed = s["x"].double()
    if s["residual"] is not None:
        summed = (summed + s["residual"].double()).to(s["dtype"]).double()
    y = summed / torch.sqrt(summed.square().sum(dim=1, keepdim=True) / cols + 1e-6) * s["weight"].double()
    q, scales = torch.empty_like(y), []
    for at in range(0, cols, 128):
        block = y[:, at:at + 128]
        scale = torch.clamp(block.abs().max(dim=1).values / E4M3_MAX, min=SMALLEST_SCALE)
        scales.append(scale)
        v = (block / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
        # e4m3: 4 significant bits from 2^-6 up, steps of 2^-9 below; ties to even
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
        q[:, at:at + 128] = torch.round(v / step) * step
    return {"rows": q, "scales": torch.stack(scales, dim=1), "sum": summed}


def _exact_product(s):
    rows, out, cols = s["case"]["rows"], s["case"]["out"], s["case"]["cols"]
    total = torch.zeros((rows, out), dtype=torch.float64, device="cuda")
    of_row = torch.arange(out, device="cuda") // 128
    step = 2048
    for at in range(0, cols, step):
        end = min(cols, at + step)
        of_col = torch.arange(at, end, device="cuda") // 128
        x = s["x"][:, at:end].double() * s["x_scales"].double()[:, of_col]
        w = s["w"][:, at:end].double() * s["w_scales"].double()[of_row][:, of_col]
        total += x @ w.t()
    return total


def _exact_append(s):
    before, rows = _sizes(s["case"])
    page = s["case"]["page"]
    seq = [b for b, r in enumerate(rows) for _ in range(r)]
    pos = [before[b] + i for b, r in enumerate(rows) for i in range(r)]
    seq, pos = torch.tensor(seq, device="cuda"), torch.tensor(pos, device="cuda")
    turn = torch.polar(torch.ones((pos.numel(), 1, s["frequencies"].numel()), dtype=torch.float64, device="cuda"),
                       (pos.double()[:, None] * s["frequencies"])[:, None, :])

    def rotated(x):
        half = x.shape[2] // 2
        z = torch.complex(x[:, :, :half].double(), x[:, :, half:].double()) * turn
        return torch.cat((z.real, z.imag), dim=2)

    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    where = s["page_table"].long()[seq, torch.div(pos, page, rounding_mode="floor")] * page + pos % page
    k_cache.flatten(0, 1)[where] = rotated(s["k"])
    v_cache.flatten(0, 1)[where] = s["v"].double()
    return {"q": rotated(s["q"]), "k_cache": k_cache, "v_cache": v_cache}


def _exact_attention(s):
    case = s["case"]
    before, rows = _sizes(case)
    group, page = case["heads"] // case["kv_heads"], case["page"]
    q_all = s["q"].reshape(case["sequences"], case["rows"], case["heads"], case["head"]).double()
    out = torch.empty_like(q_all)
    for b, length in enumerate(before):
        tokens = length + rows[b]
        pages = s["page_table"][b, :(tokens + page - 1) // page].long()
        k = s["k_cache"][pages].flatten(0, 1)[:tokens].double()
        v = s["v_cache"][pages].flatten(0, 1)[:tokens].double()
        for h in range(case["kv_heads"]):
            kh, vh = k[:, h].contiguous(), v[:, h].contiguous()
            for r in range(case["rows"]):
                n = length + r + 1
                score = q_all[b, r, h * group:(h + 1) * group] @ kh[:n].t() / math.sqrt(case["head"])
                out[b, r, h * group:(h + 1) * group] = torch.softmax(score, dim=1) @ vh[:n]
    return out[:, 0] if case["rows"] == 1 else out


def exact(case, seed):
    state = prepare(case, seed)
    return {"norm": _exact_norm, "product": _exact_product, "append": _exact_append,
            "attention": _exact_attention}[case["kind"]](state)
