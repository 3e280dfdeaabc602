"""The operators that prompts and long contexts add to a paged cache, as cases to measure.

  norm_append  queries and keys normed head by head and rotated to their positions, keys and values
               written into the pages of their sequences, in one pass
  append8      the same into pages of e4m3 values with a scale for each position and head (with the
               norms or without)
  decode8      one to eight new query rows of each sequence over such pages
  chunk        any number of new query rows of each sequence over its 16-bit pages, packed one
               sequence after another: whole prompts, chunks of them, single tokens among them
  chunk8       the same over e4m3 pages

`run` computes them either in their plain form (elementary torch operations in 32 bits, positions'
angles in 64) or, where `own` is true, through pocketlm_amd.native.  Sizes are those of the
repository's benchmark (a dense layer of 28 query and 4 key-value heads of 128) and generic ones.
16-bit values are N(0, 1); e4m3 pages hold N(0, 120) cut off at 448, as a quantizer leaves them, with
scales uniform in (4e-3, 9e-3).
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3_MAX = 448.0
SMALLEST_SCALE = 2.0 ** -126
EPS = 1e-6


def listed():
    dense = {"heads": 28, "kv_heads": 4, "head": 128}
    return [
        # one generated token: the latency of the call
        {"name": "norm_append_token", "kind": "norm_append", **dense, "sequences": 1, "rows": 1, "context": 700, "ragged": False,
         "page": 16, "pairs": 64, "interleaved": False, "norms": True, "dtype": "bf16"},
        # one step of a batch of decoding sequences
        {"name": "norm_append_batch", "kind": "norm_append", "heads": 32, "kv_heads": 8, "head": 128, "sequences": 64,
         "rows": 1, "context": 1000, "ragged": True, "page": 16, "pairs": 64, "interleaved": False, "norms": True,
         "dtype": "bf16"},
        # a few prompts of ragged lengths into an empty cache
        {"name": "norm_append_prompts", "kind": "norm_append", **dense, "sequences": 5, "rows": 1700, "context": 0,
         "ragged": True, "page": 64, "pairs": 64, "interleaved": False, "norms": True, "dtype": "fp16"},
        # one step of a batch of decoding sequences, a quarter of each head rotated, neighbours in pairs
        {"name": "append8_batch", "kind": "append8", **dense, "sequences": 64, "rows": 1, "context": 1000, "ragged": True,
         "page": 16, "pairs": 16, "interleaved": True, "norms": False, "dtype": "bf16"},
        # a few prompts of ragged lengths into an empty cache
        {"name": "append8_prompts", "kind": "append8", **dense, "sequences": 5, "rows": 1700, "context": 0, "ragged": True,
         "page": 64, "pairs": 64, "interleaved": False, "norms": True, "dtype": "bf16"},
        # one sequence, a short conversation: the latency of the call
        {"name": "decode8_short", "kind": "decode8", **dense, "sequences": 1, "rows": 1, "context": 700, "ragged": False,
         "page": 16, "dtype": "bf16"},
        # a server's batch of long conversations
        {"name": "decode8_batch", "kind": "decode8", **dense, "sequences": 48, "rows": 1, "context": 16381, "ragged": True,
         "page": 16, "dtype": "bf16"},
        # a short question after a short conversation: the latency of the call
        {"name": "chunk_question", "kind": "chunk", **dense, "sequences": 1, "rows": 37, "context": 700, "ragged": False,
         "page": 16, "dtype": "bf16"},
        # a chunk of ragged length of a few long prompts, most of which are in the cache
        {"name": "chunk_history", "kind": "chunk", **dense, "sequences": 3, "rows": 509, "context": 20000, "ragged": True,
         "page": 16, "dtype": "fp16"},
        # whole prompts
        {"name": "chunk_prompts", "kind": "chunk", **dense, "sequences": 2, "rows": 8191, "context": 0, "ragged": True,
         "page": 64, "dtype": "bf16"},
        # a short turn of each of a few conversations in a quantized cache
        {"name": "chunk8_turns", "kind": "chunk8", **dense, "sequences": 6, "rows": 24, "context": 5003, "ragged": True,
         "page": 32, "dtype": "bf16"},
        # the last chunk of a long prompt in a quantized cache
        {"name": "chunk8_history", "kind": "chunk8", **dense, "sequences": 1, "rows": 2048, "context": 30000,
         "ragged": False, "page": 64, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm_append", "append8", "decode8", "decode8", "chunk", "chunk", "chunk", "chunk8", "chunk8"])
    heads, kv_heads, head = rng.choice([(14, 2, 64), (12, 2, 128), (16, 8, 64), (32, 8, 64), (28, 4, 128), (16, 16, 64),
                                        (32, 1, 128), (8, 4, 256), (20, 5, 96), (6, 3, 80)])
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "head": head,
            "page": rng.choice([8, 16, 16, 32, 64, 100, 128, 256]), "ragged": rng.random() < 0.7,
            "dtype": rng.choice(["fp16", "bf16", "bf16"])}
    if kind in ("norm_append", "append8"):
        case.update(pairs=head // rng.choice([2, 2, 2, 4, 8]), interleaved=rng.random() < 0.3,
                    norms=kind == "norm_append" or rng.random() < 0.5)
        if rng.random() < 0.5:
            return {**case, "sequences": _log(rng, 1, 64), "rows": rng.choice([1, 1, 2, 4, 8]),
                    "context": _log(rng, 16, 2000)}
        return {**case, "sequences": rng.randint(1, 5), "rows": _log(rng, 16, 1700), "context": rng.choice([0, 0, 333])}
    if kind == "decode8":
        # at most the bytes of the largest listed cache
        context = _log(rng, 16, 32768)
        most = 48 * 16381 * 4 * 128 // (context * kv_heads * head)
        return {**case, "sequences": _log(rng, 1, max(1, min(64, most))), "rows": rng.choice([1, 1, 1, 2, 4, 8]),
                "context": context}
    # at most the products of the largest listed case, in 32 bits at most 15 GB of scores
    rows = _log(rng, 2, 8191)
    context = rows + (0 if rng.random() < 0.4 else _log(rng, 16, 32768))
    most = 7700 * 7700 * 28 * 128
    if rows * context * heads * head > most:
        rows = max(2, most // (context * heads * head))
    most //= rows * context * heads * head
    return {**case, "sequences": _log(rng, 1, max(1, min(48, most))), "rows": rows, "context": context - rows}


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
        piece = torch.randn(n, generator=g, device="cuda") * std
        flat[at:at + n] = (piece.clamp(-E4M3_MAX, E4M3_MAX) if dtype == torch.float8_e4m3fn else piece).to(dtype)
    return out


def _spread(most, count, ragged):
    """`count` sizes, the largest `most`; ragged ones go down to about half of it."""
    return [max(0, int(round(most * (1.0 - 0.5 * i / count)))) if ragged else most for i in range(count)]


def _sizes(case):
    """The tokens that each sequence has before the call, and its new rows."""
    n, kind = case["sequences"], case["kind"]
    if kind in ("chunk", "chunk8") or (kind != "decode8" and case["rows"] > 8):
        return _spread(case["context"], n, case["ragged"]), [max(1, r) for r in _spread(case["rows"], n, case["ragged"])]
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
    state = {"page_table": table.to(torch.int32).contiguous(),
             "lengths": torch.tensor(before, dtype=torch.int32, device="cuda")}
    if case["kind"] in ("append8", "decode8", "chunk8"):
        for name in ("k", "v"):
            state[name + "_cache"] = _randn(shape, g, torch.float8_e4m3fn, 120.0)
            state[name + "_scales"] = torch.rand((total, kvh, page), generator=g, device="cuda") * 5e-3 + 4e-3
    else:
        state["k_cache"], state["v_cache"] = _randn(shape, g, DTYPES[case["dtype"]]), _randn(shape, g, DTYPES[case["dtype"]])
    return state


def prepare(case, seed):
    g = _gen(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    heads, kvh, head = case["heads"], case["kv_heads"], case["head"]
    before, rows = _sizes(case)
    state = {"case": case, "dtype": dtype, **_cache(case, g, before, rows)}
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    state["row_starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    if kind == "decode8":
        q = _randn((case["sequences"], case["rows"], heads, head), g, dtype)
        state["q"] = q[:, 0] if case["rows"] == 1 else q
        return state
    if kind in ("chunk", "chunk8"):
        state["q"] = _randn((starts[-1], heads, head), g, dtype)
        return state
    # q, k and v as the fused projection leaves them: columns of one matrix
    qkv = _randn((starts[-1], (heads + 2 * kvh) * head), g, dtype)
    q, k, v = qkv.split([heads * head, kvh * head, kvh * head], dim=1)
    state["q"], state["k"], state["v"] = (t.unflatten(1, (-1, head)) for t in (q, k, v))
    pairs = case["pairs"]
    state["frequencies"] = torch.tensor([1e6 ** (-float(i) / pairs) for i in range(pairs)], dtype=torch.float64,
                                        device="cuda")
    state["q_weight"] = state["k_weight"] = None
    if case["norms"]:
        state["q_weight"] = (1.0 + 0.1 * torch.randn(head, generator=g, device="cuda")).to(dtype)
        state["k_weight"] = (1.0 + 0.1 * torch.randn(head, generator=g, device="cuda")).to(dtype)
    return state


# ---------------------------------------------------------------- the plain forms

def _row_places(s):
    """The sequence and the position of each new row."""
    starts = s["row_starts"].long()
    n = torch.arange(int(s["q"].shape[0]), device="cuda")
    seq = torch.searchsorted(starts, n, right=True) - 1
    return seq, s["lengths"].long()[seq] + n - starts[seq]


def _turned(x, weight, cos, sin, interleaved):
    """Heads normed (with a weight) and rotated, in 32 bits."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(dim=2, keepdim=True) + EPS) * weight.float()
    pairs = cos.shape[2]
    y, rest = x[:, :, :2 * pairs], x[:, :, 2 * pairs:]
    if interleaved:
        a, b = y[:, :, 0::2], y[:, :, 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=3).flatten(2)
    else:
        a, b = y[:, :, :pairs], y[:, :, pairs:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=2)
    return torch.cat((y, rest), dim=2)


def _append(s):
    case = s["case"]
    seq, pos = _row_places(s)
    angle = pos.double()[:, None] * s["frequencies"][None, :]
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    page = case["page"]
    at, slot = s["page_table"][seq, pos // page].long(), pos % page
    q = _turned(s["q"], s["q_weight"], cos, sin, case["interleaved"]).to(s["dtype"])
    k = _turned(s["k"], s["k_weight"], cos, sin, case["interleaved"])
    out = {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if case["kind"] == "norm_append":
        s["k_cache"][at, slot] = k.to(s["dtype"])
        s["v_cache"][at, slot] = s["v"]
        return out
    for name, x in (("k", k), ("v", s["v"].float())):
        scale = (x.abs().amax(dim=2) / E4M3_MAX).clamp(min=SMALLEST_SCALE)
        held = (x / scale[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        s[name + "_cache"].view(torch.uint8)[at, slot] = held.view(torch.uint8)
        s[name + "_scales"][at, :, slot] = scale
        out[name + "_scales"] = s[name + "_scales"]
    return out


def _attention(s):
    case = s["case"]
    page, kvh, head, rows = case["page"], case["kv_heads"], case["head"], case["rows"]
    group, n = case["heads"] // kvh, case["sequences"]
    length = s["page_table"].shape[1] * page
    at = torch.arange(length, device="cuda")
    pages, slots = s["page_table"].long()[:, at // page], at % page

    def gathered(name):
        held = s[name + "_cache"]
        if held.dtype != torch.float8_e4m3fn:
            return held[pages, slots].float()
        values = held.view(torch.uint8)[pages, slots].view(torch.float8_e4m3fn).float()
        return values * s[name + "_scales"][pages, :, slots][:, :, :, None]

    k = gathered("k").permute(0, 2, 3, 1).contiguous()  # [n, kvh, head, length]
    v = gathered("v").permute(0, 2, 1, 3).contiguous()  # [n, kvh, length, head]
    # queries padded to as many rows a sequence
    starts = s["row_starts"].long()
    row = torch.arange(rows, device="cuda")
    there = row[None, :] < (starts[1:] - starts[:-1])[:, None]
    flat = s["q"].reshape(-1, case["heads"], head)
    q = flat[(starts[:-1, None] + row[None, :]).clamp(max=flat.shape[0] - 1)].float()
    q = q.view(n, rows, kvh, group, head).permute(0, 2, 1, 3, 4).reshape(n, kvh, rows * group, head)
    seen = s["lengths"].long()[:, None] + 1 + row[None, :]
    hidden = at[None, None, :] >= seen[:, :, None]
    scores = torch.matmul(q, k).mul_(1.0 / math.sqrt(head)).view(n, kvh, rows, group, length)
    scores.masked_fill_(hidden[:, None, :, None, :], -math.inf)
    p = scores.sub_(scores.amax(dim=4, keepdim=True)).exp_().view(n, kvh, rows * group, length)
    out = torch.matmul(p, v) / p.sum(dim=3, keepdim=True)
    out = out.view(n, kvh, rows, group, head).permute(0, 2, 1, 3, 4).reshape(n, rows, kvh * group, head).to(s["dtype"])
    return out[there].view(s["q"].shape)


# ---------------------------------------------------------------- a pass

def _own(s):
    from pocketlm_amd import native

    case = s["case"]
    kind = case["kind"]
    where = (s["page_table"], s["lengths"])
    if kind == "norm_append":
        q = native.kv_paged_norm_append(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["k_cache"], s["v_cache"],
                                        *where, rms_eps=EPS, row_starts=None if case["rows"] <= 8 else s["row_starts"],
                                        rope_frequencies=s["frequencies"], interleaved=case["interleaved"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if kind == "chunk":
        return native.kv_paged_attention_chunk(s["q"], s["k_cache"], s["v_cache"], *where, s["row_starts"])
    held = (s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"])
    if kind == "append8":
        q = native.kv_paged_append_e4m3(s["q"], s["k"], s["v"], *held, *where, q_norm_weight=s["q_weight"],
                                        k_norm_weight=s["k_weight"], rms_eps=EPS,
                                        row_starts=None if case["rows"] <= 8 else s["row_starts"],
                                        rope_frequencies=s["frequencies"], interleaved=case["interleaved"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"], "k_scales": s["k_scales"],
                "v_scales": s["v_scales"]}
    if kind == "decode8":
        return native.kv_paged_attention_decode_e4m3(s["q"], *held, *where)
    return native.kv_paged_attention_chunk_e4m3(s["q"], *held, *where, s["row_starts"])


def run(state):
    if own:
        return _own(state)
    return _append(state) if state["case"]["kind"] in ("norm_append", "append8") else _attention(state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    before, rows = _sizes(case)
    heads, kvh, head, kind = case["heads"], case["kv_heads"], case["head"], case["kind"]
    held = 2 * head if kind in ("norm_append", "chunk") else head + 4  # bytes of a position's head in a cache
    new = sum(rows)
    if kind in ("norm_append", "append8"):
        moved = new * (heads + 2 * kvh) * head * 2 + new * heads * head * 2 + new * 2 * kvh * held
        return {"bytes": moved, "flops": new * (heads + kvh) * head * (6 if case["norms"] else 3)}
    seen = sum(b + r for b, r in zip(before, rows))
    pairs = sum(r * (b + (r + 1) / 2) for b, r in zip(before, rows))
    return {"bytes": 2 * seen * kvh * held + 2 * new * heads * head * 2, "flops": 4 * pairs * heads * head}


# ---------------------------------------------------------------- the definition in 64 bits

def _exact_append(s):
    case = s["case"]
    before, rows = _sizes(case)
    page, pairs = case["page"], case["pairs"]
    seq = torch.tensor([b for b, r in enumerate(rows) for _ in range(r)], device="cuda")
    pos = torch.tensor([before[b] + i for b, r in enumerate(rows) for i in range(r)], device="cuda")
    turn = torch.polar(torch.ones((pos.numel(), 1, pairs), dtype=torch.float64, device="cuda"),
                       (pos.double()[:, None] * s["frequencies"])[:, None, :])

    def definition(x, weight):
        y = x.double()
        if weight is not None:
            y = y / torch.sqrt(y.square().sum(dim=2, keepdim=True) / y.shape[2] + EPS) * weight.double()
        else:
            y = y.clone()
        first = slice(0, 2 * pairs, 2) if case["interleaved"] else slice(0, pairs)
        second = slice(1, 2 * pairs, 2) if case["interleaved"] else slice(pairs, 2 * pairs)
        z = torch.complex(y[:, :, first].contiguous(), y[:, :, second].contiguous()) * turn
        y[:, :, first], y[:, :, second] = z.real, z.imag
        return y

    where = s["page_table"].long()[seq, torch.div(pos, page, rounding_mode="floor")] * page + pos % page
    out = {"q": definition(s["q"], s["q_weight"])}
    for name, y in (("k", definition(s["k"], s["k_weight"])), ("v", s["v"].double())):
        cache = s[name + "_cache"].double()
        if case["kind"] == "append8":
            scale = torch.clamp(y.abs().max(dim=2).values / E4M3_MAX, min=SMALLEST_SCALE)
            u = (y / scale[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
            # e4m3: 4 significant bits from 2^-6 up, steps of 2^-9 below; ties to even
            step = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3)
            y = torch.round(u / step) * step
            scales = s[name + "_scales"].double().transpose(1, 2).contiguous()
            scales.view(-1, scales.shape[2])[where] = scale
            out[name + "_scales"] = scales.transpose(1, 2).contiguous()
        cache.flatten(0, 1)[where] = y
        out[name + "_cache"] = cache
    return out


def _exact_attention(s):
    case = s["case"]
    before, rows = _sizes(case)
    group, page = case["heads"] // case["kv_heads"], case["page"]
    flat = s["q"].reshape(-1, case["heads"], case["head"]).double()
    out = torch.empty_like(flat)
    first = 0
    for b, length in enumerate(before):
        tokens = length + rows[b]
        pages = s["page_table"][b, :(tokens + page - 1) // page].long()
        for h in range(case["kv_heads"]):
            kv = []
            for name in ("k", "v"):
                x = s[name + "_cache"][pages][:, :, h].double() if s[name + "_cache"].dtype != torch.float8_e4m3fn else \
                    s[name + "_cache"].view(torch.uint8)[pages][:, :, h].contiguous().view(torch.float8_e4m3fn).double() \
                    * s[name + "_scales"][pages][:, h].double()[:, :, None]
                kv.append(x.flatten(0, 1)[:tokens].contiguous())
            # a few rows at a time
            for at in range(0, rows[b], 1024):
                r = min(1024, rows[b] - at)
                n = length + at + r
                q = flat[first + at:first + at + r, h * group:(h + 1) * group].transpose(0, 1).contiguous()
                score = torch.matmul(q, kv[0][:n].t().contiguous()) / math.sqrt(case["head"])
                late = torch.arange(n, device="cuda")[None, :] > length + at + torch.arange(r, device="cuda")[:, None]
                weight = torch.softmax(score.masked_fill_(late[None], -math.inf), dim=2)
                out[first + at:first + at + r, h * group:(h + 1) * group] = torch.matmul(weight, kv[1][:n]).transpose(0, 1)
        first += rows[b]
    return out.view(s["q"].shape)


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_append(state) if case["kind"] in ("norm_append", "append8") else _exact_attention(state)
