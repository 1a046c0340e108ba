"""Operators of a cache whose older pages are held in 8 bits, and of beam search over it.

Five operators: pages of keys and values to 8 bits (a scale for each 8 tokens of a head) and back, attention of single
tokens over such pages and the bf16 pages after them, attention of spans of tokens over the same, beam search's
selection over beams and vocabulary, and the copies of pages that its reordering of the beams needs.
Each in its plain form (elementary torch operations in 32 bits) and through the framework's entry points.
"""

import math

import torch

own = False

PAGE = 16
BLOCK = 8  # tokens that share a scale
VOCAB = 128256


def listed():
    return [
        # the finished chunk of one sequence: latency
        {"name": "quantize_64x8x128", "op": "quantize", "pages": 64, "hkv": 8, "d": 128, "ragged": False},
        # the finished chunks of 64 sequences at once
        {"name": "quantize_4096x8x128", "op": "quantize", "pages": 4096, "hkv": 8, "d": 128, "ragged": False},
        # a short prompt of a small model of 12 heads, one sequence: latency
        {"name": "decode_1x512_12h", "op": "decode", "batch": 1, "context": 512, "chunk": 128, "hq": 12, "hkv": 12,
         "d": 64, "lens": "full"},
        # a decode step's layer of the 8B architecture, 8 sequences
        {"name": "decode_8x8192", "op": "decode", "batch": 8, "context": 8192, "chunk": 1024, "hq": 32, "hkv": 8,
         "d": 128, "lens": "full"},
        # the largest: 64 sequences
        {"name": "decode_64x8192", "op": "decode", "batch": 64, "context": 8192, "chunk": 1024, "hq": 32, "hkv": 8,
         "d": 128, "lens": "full"},
        # requests of all lengths, some of them empty, every page in 8 bits
        {"name": "decode_33x5000_ragged", "op": "decode", "batch": 33, "context": 5000, "chunk": 0, "hq": 8, "hkv": 4,
         "d": 64, "lens": "ragged"},
        # a chunk of two prompts, 7168 tokens into them
        {"name": "prefill_2x1024_8192", "op": "prefill", "batch": 2, "span": 1024, "context": 8192, "chunk": 1024,
         "hq": 32, "hkv": 8, "d": 128, "lens": "full"},
        # short spans of ragged requests (the rest of a prompt, drafted tokens)
        {"name": "prefill_5x200_3000", "op": "prefill", "batch": 5, "span": 200, "context": 3000, "chunk": 256,
         "hq": 8, "hkv": 4, "d": 64, "lens": "ragged"},
        # one request with 4 beams
        {"name": "beam_1x4", "op": "beam", "batch": 1, "beams": 4, "select": 4, "vocab": VOCAB, "type": "bf16",
         "finished": False},
        # 16 requests with 8 beams, twice as many candidates as beams, an odd vocabulary, some beams finished
        {"name": "beam_16x8_odd", "op": "beam", "batch": 16, "beams": 8, "select": 16, "vocab": 50001, "type": "fp32",
         "finished": True},
        # the pages that 4 beams of a small model write to
        {"name": "reorder_4_12l", "op": "reorder", "rows": 4, "layers": 12, "hkv": 12, "d": 64},
        # 8 requests with 8 beams, every layer of the 8B architecture
        {"name": "reorder_64_32l", "op": "reorder", "rows": 64, "layers": 32, "hkv": 8, "d": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "decode", "decode", "decode", "prefill", "prefill", "beam", "beam", "reorder"])
    hkv, group, d = rng.choice([1, 2, 4, 8, 12]), rng.choice([1, 2, 4, 8]), rng.choice([64, 128])
    if op == "quantize":
        return {"op": op, "pages": _log(rng, 1, 4096), "hkv": min(hkv, 8), "d": d, "ragged": rng.choice([False, True])}
    if op == "decode":
        hkv = min(hkv, 8) if d == 128 else hkv
        context = _log(rng, 1, 131072)
        most = max(1, 64 * 8192 * 8 * 128 // (context * hkv * d))
        return {"op": op, "batch": _log(rng, 1, min(most, 256)), "context": context,
                "chunk": rng.choice([0, 16, 128, 1024]), "hq": hkv * group, "hkv": hkv, "d": d,
                "lens": rng.choice(["full", "ragged"])}
    if op == "prefill":
        chunk, context = rng.choice([0, 256, 1024]), _log(rng, 16, 16384)
        span = min(_log(rng, 1, 1024), context, chunk or 1024)
        heads = hkv * group
        most = max(1, 2 * 1024 * 32 * 8192 // (span * heads * context))
        return {"op": op, "batch": _log(rng, 1, min(most, 16)), "span": span, "context": context, "chunk": chunk,
                "hq": heads, "hkv": hkv, "d": d, "lens": rng.choice(["full", "ragged"])}
    if op == "beam":
        beams, vocab = _log(rng, 1, 16), _log(rng, 100, 200000)
        return {"op": op, "batch": _log(rng, 1, max(1, min(64, 8_000_000 // (beams * vocab)))), "beams": beams,
                "select": min(beams * rng.choice([1, 2]), vocab), "vocab": vocab, "type": rng.choice(["bf16", "fp32"]),
                "finished": rng.choice([False, True])}
    return {"op": op, "rows": _log(rng, 1, 64), "layers": _log(rng, 1, 32), "hkv": min(hkv, 8), "d": d}


# ---------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _rows(shape, g):
    """Keys or values as a cache holds them: normal, a few of a head's columns larger than the rest."""
    x = torch.randn(shape, generator=g, device="cuda")
    big = torch.rand(shape[-2:], generator=g, device="cuda") < 0.02
    return x.mul_(torch.where(big, 5.0, 1.0)).bfloat16()


def _quantized(x):
    """(codes int8, scales fp32 [pages, 2, Hkv]) of pages [pages, 16, Hkv, D]."""
    y = x.float().view(x.shape[0], PAGE // BLOCK, BLOCK, *x.shape[2:])
    scale = y.abs().amax((2, 4)) / 127
    s = scale[:, :, None, :, None]
    return torch.where(s == 0, 0, torch.round(y / s)).to(torch.int8).view(x.shape), scale


def _spread(B, g):
    """B numbers between 0 and 1, the same in every order that a seed puts them in."""
    return (torch.randperm(B, generator=g, device="cuda").double() + 0.5) / B


def _lengths(case, g):
    """(tokens in the cache, new tokens among them) of each request."""
    B, ctx = case["batch"], case["context"]
    u = _spread(B, g)
    if case["lens"] == "full":
        n = (ctx * (1 + u) / 2).ceil().long()
    else:
        n = torch.exp(u * math.log(ctx + 1)).long()
        if case["op"] == "decode" and B > 4:
            n[:2] = torch.arange(2, device="cuda")  # an empty request, and one of a single token
    if case["op"] == "decode":
        return n.clamp(max=ctx), None
    span = torch.full_like(n, case["span"])
    if case["lens"] == "ragged":  # some of them without a new token
        span = torch.exp(_spread(B, g) * math.log(case["span"] + 1)).long() - (_spread(B, g) < 0.2).long()
    return n.clamp(max=ctx).maximum(span), span


def _cache_inputs(case, seed):
    """Tables over shuffled pages, the older ones in 8 bits and those of the last one or two chunks in bf16."""
    g = _gen(seed)
    B, C, hkv, d = case["batch"], case["chunk"], case["hkv"], case["d"]
    n, span = _lengths(case, g)
    W = -(-case["context"] // PAGE)
    pages = (n + PAGE - 1) // PAGE
    if C:
        older = ((n - 1).clamp(min=0) // C * C - C).clamp(min=0) // PAGE
    else:
        older = pages
    col = torch.arange(W, device="cuda")
    old, new = col < older[:, None], (col >= older[:, None]) & (col < pages[:, None])
    n_old, n_new = int(old.sum()), int(new.sum())
    table = torch.zeros((B, W), dtype=torch.int64, device="cuda")
    table[old] = torch.randperm(n_old, generator=g, device="cuda")
    table[new] = torch.randperm(n_new, generator=g, device="cuda")
    k, ks = _quantized(_rows((n_old + 1, PAGE, hkv, d), g))
    v, vs = _quantized(_rows((n_old + 1, PAGE, hkv, d), g))
    s = {"case": case, "k": k, "ks": ks, "v": v, "vs": vs, "table": table.int(), "older": older.int(),
         "seq_k": n.int(), "pool_k": _rows((n_new + 1, PAGE, hkv, d), g), "pool_v": _rows((n_new + 1, PAGE, hkv, d), g)}
    if case["op"] == "decode":
        s["q"] = _rows((B, case["hq"], d), g)
    else:
        s["cu_q"] = torch.cat((span.new_zeros(1), span.cumsum(0))).int()
        s["q"] = _rows((int(span.sum()), case["hq"], d), g)
    return s


def _quantize_inputs(case, seed):
    g, N = _gen(seed), case["pages"]
    shape = (N + 3, PAGE, case["hkv"], case["d"])
    s = {"case": case, "pool_k": _rows(shape, g), "pool_v": _rows(shape, g),
         "pages": torch.randperm(N + 3, generator=g, device="cuda")[:N].int(),
         "out_pages": torch.randperm(N, generator=g, device="cuda").int()}
    # pages of a sequence's end hold fewer than 16 tokens
    s["tokens"] = torch.randint(0, PAGE + 1, (N,), generator=g, device="cuda").int() if case["ragged"] else None
    return s


def _beam_inputs(case, seed):
    g, B, K, V = _gen(seed), case["batch"], case["beams"], case["vocab"]
    logits = torch.randn((B * K, V), generator=g, device="cuda") * 2.5
    if case["type"] == "bf16":
        logits = logits.bfloat16()
    scores = -torch.rand((B, K), generator=g, device="cuda") * 6 - 10
    s = {"case": case, "logits": logits, "scores": scores.sort(descending=True).values, "finished": None, "eos": -1}
    if case["finished"]:
        s["finished"], s["eos"] = torch.rand((B, K), generator=g, device="cuda") < 0.25, V // 3
    return s


def _reorder_inputs(case, seed):
    g, R, L = _gen(seed), case["rows"], case["layers"]
    stride = 2 * R + 1  # a page for each row to write to, as many free ones, a scratch page
    shape = (L * stride, PAGE, case["hkv"], case["d"])
    ids = torch.randperm(2 * R, generator=g, device="cuda")
    parents = torch.randint(0, R, (R,), generator=g, device="cuda")
    return {"case": case, "pool_k": _rows(shape, g), "pool_v": _rows(shape, g), "src": ids[:R][parents].int(),
            "dst": ids[R:].int(), "stride": stride}


_INPUTS = {"quantize": _quantize_inputs, "decode": _cache_inputs, "prefill": _cache_inputs, "beam": _beam_inputs,
           "reorder": _reorder_inputs}


def prepare(case, seed):
    s = _INPUTS[case["op"]](case, seed)
    if own:
        from lastkv_b200 import ops

        if case["op"] == "quantize":
            s["cache"] = ops.PagesQ8.empty(case["pages"], case["hkv"], case["d"], device="cuda")
            s["back_k"], s["back_v"] = (torch.empty((case["pages"], PAGE, case["hkv"], case["d"]), dtype=torch.bfloat16,
                                                    device="cuda") for _ in range(2))
            s["all"] = torch.arange(case["pages"], dtype=torch.int32, device="cuda")
        elif case["op"] in ("decode", "prefill"):  # the cache as the program filled it, and the step's workspaces
            s["cache"] = ops.PagesQ8.from_codes(s.pop("k"), s.pop("v"), s.pop("ks"), s.pop("vs"))
            W = s["table"].shape[1]
            if case["op"] == "decode":
                s["workspace"] = ops.Workspace.for_decode(case["batch"], case["hq"], case["d"], W)
            else:
                s["stage"] = ops.StageQ8.empty(case["batch"], W, case["hkv"], case["d"], device="cuda")
    return s


# ---------------------------------------------------------------- plain forms


def _quantize_plain(s):
    out = {}
    for name in ("k", "v"):
        x = s["pool_" + name][s["pages"].long()]
        if s["tokens"] is not None:
            tok = torch.arange(PAGE, device=x.device)
            x = torch.where((tok < s["tokens"][:, None])[:, :, None, None], x, 0)
        codes, scale = _quantized(x)
        y = codes.float() * scale.repeat_interleave(BLOCK, 1)[..., None]
        out[name], out[name + "_scale"] = torch.empty_like(x), torch.empty_like(scale)
        out[name][s["out_pages"].long()] = y.bfloat16()
        out[name + "_scale"][s["out_pages"].long()] = scale
    return out


def _gathered(s, name):
    """Every row's keys or values, fp32 [B, W * 16, Hkv, D]."""
    t = s["table"].long()
    old = (torch.arange(t.shape[1], device=t.device) < s["older"][:, None])
    ids = torch.where(old, t, 0)
    y = s[name][ids].float().mul_(s[name + "s"].repeat_interleave(BLOCK, 1)[ids][..., None])
    y = torch.where(old[:, :, None, None, None], y, s["pool_" + name][torch.where(old, 0, t)].float())
    return y.flatten(1, 2)


def _softmax_rows(scores, seen):
    """Softmax of the last axis over the keys that a row sees; rows that see none are zero."""
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0, top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, 1, total)


def _attend_plain(s):
    c = s["case"]
    B, hkv, d, G = c["batch"], c["hkv"], c["d"], c["hq"] // c["hkv"]
    key = torch.arange(s["table"].shape[1] * PAGE, device="cuda")
    n = s["seq_k"].long()
    if c["op"] == "decode":
        q, last = s["q"].float().view(B, 1, hkv, G, d), n[:, None] - 1
    else:  # the rows' spans, side by side
        cu, top = s["cu_q"].long(), c["span"]
        t = torch.arange(top, device="cuda")
        lq = (cu[1:] - cu[:-1])[:, None]
        at = (cu[:-1, None] + t).clamp(max=max(s["q"].shape[0] - 1, 0))
        q = s["q"].float()[at].view(B, top, hkv, G, d)
        last = torch.where(t < lq, n[:, None] - lq + t, -1)
    scores = torch.einsum("bthgd,bkhd->bthgk", q * d ** -0.5, _gathered(s, "k"))
    seen = (key <= last[:, :, None]) & (key < n[:, None, None])
    p = _softmax_rows(scores, seen[:, :, None, None])
    out = torch.einsum("bthgk,bkhd->bthgd", p, _gathered(s, "v")).reshape(B, -1, c["hq"], d)
    return (out[:, 0] if c["op"] == "decode" else out[t < lq]).bfloat16()


def _beam_plain(s):
    """In 64 bits: totals of different beams lie close together."""
    c = s["case"]
    B, K, V, n = c["batch"], c["beams"], c["vocab"], c["select"]
    x = s["logits"].double().view(B, K, V)
    top = x.amax(-1, keepdim=True)
    total = x - (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))) + s["scores"].double()[..., None]
    done = s["finished"]
    if done is not None:  # a finished beam goes on as it is, with the one token that says so
        alone = torch.where(torch.arange(V, device="cuda") == s["eos"], s["scores"].double()[..., None], -math.inf)
        total = torch.where(done[..., None], alone, total)
    best, at = total.view(B, K * V).sort(dim=-1, descending=True, stable=True)
    best, at = best[:, :n], at[:, :n]
    beam, token = torch.div(at, V, rounding_mode="floor"), at % V
    ended = token == s["eos"]
    return {"scores": best.float(), "rows": beam + torch.arange(B, device="cuda")[:, None] * K, "tokens": token,
            "finished": ended if done is None else ended | done.gather(1, beam)}


def _reorder_plain(s):
    base = (torch.arange(s["case"]["layers"], device="cuda") * s["stride"])[:, None]
    for pool in (s["pool_k"], s["pool_v"]):
        pool[base + s["dst"].long()] = pool[base + s["src"].long()]
    return s["pool_k"], s["pool_v"]


# ---------------------------------------------------------------- the framework's


def _quantize_own(s):
    from lastkv_b200 import ops

    ops.quantize_pages(s["pool_k"], s["pool_v"], s["pages"], s["cache"], s["out_pages"], tokens=s["tokens"])
    ops.dequantize_pages(s["cache"], s["all"], s["back_k"], s["back_v"], s["all"])
    ks, vs = s["cache"].token_scales()
    return {"k": s["back_k"], "k_scale": ks, "v": s["back_v"], "v_scale": vs}


def _attend_own(s):
    from lastkv_b200 import ops

    if s["case"]["op"] == "decode":
        return ops.decode_paged_q8(s["q"], s["cache"], s["table"], s["seq_k"], num_q8=s["older"], pool_k=s["pool_k"],
                                   pool_v=s["pool_v"], workspace=s["workspace"])
    return ops.prefill_paged_q8(s["q"], s["cache"], s["table"], s["seq_k"], s["cu_q"], s["case"]["span"],
                                num_q8=s["older"], pool_k=s["pool_k"], pool_v=s["pool_v"], stage=s["stage"])


def _beam_own(s):
    from lastkv_b200 import ops

    r = ops.beam_select(s["logits"], s["scores"], select=s["case"]["select"], finished=s["finished"],
                        eos_token=s["eos"])
    return {"scores": r.scores, "rows": r.rows, "tokens": r.tokens, "finished": r.finished}


def _reorder_own(s):
    from lastkv_b200 import ops

    ops.reorder_pages((s["pool_k"], s["pool_v"]), s["src"], s["dst"], layers=s["case"]["layers"],
                      layer_stride=s["stride"])
    return s["pool_k"], s["pool_v"]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"quantize": _quantize_own, "decode": _attend_own, "prefill": _attend_own, "beam": _beam_own,
                "reorder": _reorder_own}[op](state)
    return {"quantize": _quantize_plain, "decode": _attend_plain, "prefill": _attend_plain, "beam": _beam_plain,
            "reorder": _reorder_plain}[op](state)


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    if case["op"] == "beam":
        n = case["batch"] * case["beams"] * case["vocab"]
        return {"bytes": n * (2 if case["type"] == "bf16" else 4) + 24 * case["batch"] * case["select"], "flops": 4 * n}
    row = case["hkv"] * case["d"]  # a token's keys (or values)
    if case["op"] == "quantize":
        tokens = case["pages"] * PAGE
        return {"bytes": tokens * row * 2 * (2 + 1 + 1 + 2), "flops": 6 * tokens * row * 2}
    if case["op"] == "reorder":
        return {"bytes": 2 * 2 * case["rows"] * case["layers"] * PAGE * row * 2, "flops": 0}
    B, ctx, C = case["batch"], case["context"], case["chunk"]
    # the mean length, as _lengths draws it
    n = 0.75 * ctx if case["lens"] == "full" else ctx / math.log(ctx + 2)
    recent = min(n, 1.5 * C)
    bytes_ = B * row * 2 * ((n - recent) * (1 + 4 / (BLOCK * case["d"])) + recent * 2)
    if case["op"] == "decode":
        return {"bytes": int(bytes_ + B * case["hq"] * case["d"] * 4), "flops": int(4 * B * n * case["hq"] * case["d"])}
    span = case["span"] if case["lens"] == "full" else case["span"] / math.log(case["span"] + 2)
    span = min(span, n)
    return {"bytes": int(bytes_ + B * span * case["hq"] * case["d"] * 4),
            "flops": int(4 * B * span * (n - span / 2) * case["hq"] * case["d"])}


# ---------------------------------------------------------------- the definitions in 64 bits


def _exact_quantize(s):
    out = {}
    for name in ("k", "v"):
        x = s["pool_" + name].double()[s["pages"].long()]
        if s["tokens"] is not None:
            x *= (torch.arange(PAGE, device="cuda")[None] < s["tokens"][:, None])[..., None, None]
        out[name], out[name + "_scale"] = torch.zeros_like(x), torch.zeros(x.shape[0], 2, x.shape[2]).double().cuda()
        for half in range(2):
            part = x[:, half * BLOCK: (half + 1) * BLOCK]
            step = part.abs().transpose(1, 2).flatten(2).max(-1).values / 127.0
            unit = step.clamp(min=1e-300)[:, None, :, None]
            out[name][s["out_pages"].long(), half * BLOCK: (half + 1) * BLOCK] = torch.round(part / unit) * unit
            out[name + "_scale"][s["out_pages"].long(), half] = step
    return out


def _exact_attend(s):
    c = s["case"]
    G, n = c["hq"] // c["hkv"], s["seq_k"].tolist()
    cu = list(range(c["batch"] + 1)) if c["op"] == "decode" else s["cu_q"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(c["batch"]):
        if not n[b] or cu[b] == cu[b + 1]:
            continue
        pages, m = -(-n[b] // PAGE), int(s["older"][b])
        ids = s["table"][b].long()
        kv = []
        for name in ("k", "v"):
            scale = s[name + "s"][ids[:m]].double()[:, :, None, :, None]
            old = (s[name][ids[:m]].double().view(m, 2, BLOCK, c["hkv"], c["d"]) * scale).view(m * PAGE, c["hkv"], c["d"])
            new = s["pool_" + name][ids[m:pages]].double().flatten(0, 1)
            kv.append(torch.cat((old, new))[: n[b]].transpose(0, 1))
        lq = cu[b + 1] - cu[b]
        late = torch.arange(n[b], device="cuda")[None] > torch.arange(n[b] - lq, n[b], device="cuda")[:, None]
        for h in range(c["hq"]):
            x = s["q"][cu[b]: cu[b + 1], h].double() @ kv[0][h // G].T / math.sqrt(c["d"])
            out[cu[b]: cu[b + 1], h] = torch.softmax(x.masked_fill_(late, -math.inf), -1) @ kv[1][h // G]
    return out


def _exact_beam(s):
    c = s["case"]
    K, n = c["beams"], c["select"]
    best = []
    for b in range(c["batch"]):
        rows = torch.log_softmax(s["logits"][b * K: (b + 1) * K].double(), -1) + s["scores"][b].double()[:, None]
        if s["finished"] is not None:
            done = s["finished"][b]
            rows[done] = -math.inf
            rows[done, s["eos"]] = s["scores"][b][done].double()
        best.append(rows.flatten().topk(n).values)
    return {"scores": torch.stack(best), "rows": None, "tokens": None, "finished": None}


def exact(case, seed):
    if case["op"] == "reorder":
        return None  # copies
    s = _INPUTS[case["op"]](case, seed)
    if case["op"] == "quantize":
        return _exact_quantize(s)
    return _exact_beam(s) if case["op"] == "beam" else _exact_attend(s)
