"""Operators of a decode or prefill step with 4-bit weights and 8-bit activations.

Three operators: rows to int8 with group scales (RMSNorm with the residual's addition, SiLU-and-mul, or the rows
themselves), products with 4-bit weights and group scales, and a step's block tables and slot maps from request lengths.
Each in its plain form (elementary torch operations in 32 bits) and through the framework's entry points.
"""

import math

import torch

own = False

PAGE = 16


def listed():
    return [
        # one token's hidden state before the q/k/v projection of the 8B architecture: launch latency
        {"name": "norm_1x4096", "op": "rows", "mode": "norm", "rows": 1, "cols": 4096, "group": 128, "pad": 0},
        # the gate | up products of a decode batch of 8, on their way into the down projection
        {"name": "silu_8x14336", "op": "rows", "mode": "silu", "rows": 8, "cols": 14336, "group": 128, "pad": 0},
        # a prefill call of 2048 tokens
        {"name": "norm_2048x4096", "op": "rows", "mode": "norm", "rows": 2048, "cols": 4096, "group": 128, "pad": 0},
        # attention outputs that are a slice of wider rows, an odd width, the smallest groups
        {"name": "plain_1000x1544", "op": "rows", "mode": "plain", "rows": 1000, "cols": 1544, "group": 32, "pad": 24},
        # a single token through the q | k | v projection
        {"name": "q8_1x6144x4096", "op": "w4", "act": "int8", "tokens": 1, "n": 6144, "k": 4096, "group": 128},
        # a decode batch of 8 through gate | up, the largest weight of a layer
        {"name": "q8_8x28672x4096", "op": "w4", "act": "int8", "tokens": 8, "n": 28672, "k": 4096, "group": 128},
        # a decode batch of 8 through the down projection, bf16 activations
        {"name": "bf16_8x4096x14336", "op": "w4", "act": "bf16", "tokens": 8, "n": 4096, "k": 14336, "group": 128},
        # a few short requests together, an odd weight, groups that end inside a block of columns
        {"name": "bf16_33x1003x1544", "op": "w4", "act": "bf16", "tokens": 33, "n": 1003, "k": 1544, "group": 64},
        # prefill calls of 2048 tokens: gate | up with int8 rows, the output projection with bf16 rows
        {"name": "q8_2048x28672x4096", "op": "w4", "act": "int8", "tokens": 2048, "n": 28672, "k": 4096, "group": 128},
        {"name": "bf16_2048x4096x4096", "op": "w4", "act": "bf16", "tokens": 2048, "n": 4096, "k": 4096, "group": 128},
        # a decode step of 8 requests near 8192 tokens (the 8B architecture's 32 layers)
        {"name": "plan_decode_8", "op": "plan", "kind": "decode", "batch": 8, "context": 8192, "layers": 32,
         "chunk": 1024, "padded": 0},
        # spans of many requests over a long context, some of them at a chunk's start
        {"name": "plan_spans_64", "op": "plan", "kind": "spans", "batch": 64, "context": 131072, "layers": 32,
         "chunk": 1024, "padded": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rows", "rows", "w4", "w4", "w4", "plan"])
    if op == "rows":
        return {"op": op, "mode": rng.choice(["norm", "silu", "plain"]), "rows": _log(rng, 1, 3000),
                "cols": 8 * _log(rng, 8, 1792), "group": rng.choice([32, 64, 128]), "pad": 8 * rng.choice([0, 0, 1, 5])}
    if op == "w4":
        n, k = _log(rng, 40, 28672), 8 * _log(rng, 8, 1792)
        most = min(2048, max(1, 2048 * 28672 * 4096 // (n * k)))
        return {"op": op, "act": rng.choice(["int8", "bf16"]), "tokens": _log(rng, 1, most), "n": n, "k": k,
                "group": rng.choice([32, 64, 128])}
    chunk, layers = rng.choice([256, 512, 1024]), rng.choice([4, 12, 32])
    kind = rng.choice(["decode", "spans"])
    context = _log(rng, 2 * chunk, 131072)
    batch = _log(rng, 1, max(1, min(256, 64 * 131072 * 32 // (context * layers))))
    return {"op": op, "kind": kind, "batch": batch, "context": context, "layers": layers, "chunk": chunk,
            "padded": rng.choice([0, 0, 3]) if kind == "decode" else 0}


# ---------------------------------------------------------------- inputs


def _gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(int(seed))


def _activations(shape, g, spread=1.0):
    """Rows as a transformer's stream has them: normal, a few columns much larger than the rest."""
    x = torch.randn(shape, generator=g, device="cuda") * spread
    big = torch.rand(shape[-1], generator=g, device="cuda") < 0.01
    return torch.where(big, x * 12, x)


def _strided(x, pad):
    """bf16 rows; with `pad`, a slice of wider rows."""
    if not pad:
        return x.bfloat16()
    wide = torch.zeros((x.shape[0], x.shape[1] + pad), dtype=torch.bfloat16, device=x.device)
    wide[:, : x.shape[1]] = x
    return wide[:, : x.shape[1]]


def _rows_inputs(case, seed):
    g, T, H = _gen(seed), case["rows"], case["cols"]
    s = {"case": case, "eps": 1e-5}
    if case["mode"] == "silu":
        s["x"] = _strided(torch.randn((T, 2 * H), generator=g, device="cuda") * 1.5, case["pad"])
        return s
    s["x"] = _strided(_activations((T, H), g), case["pad"])
    if case["mode"] == "norm":
        s["residual"] = _strided(_activations((T, H), g, 3.0), case["pad"])
        s["weight"] = (torch.rand(H, generator=g, device="cuda") + 0.5).bfloat16()
    return s


def _w4_inputs(case, seed):
    g, T, N, K, G = _gen(seed), case["tokens"], case["n"], case["k"], case["group"]
    # codes as a checkpoint holds them: two 4-bit codes u (value u - 8) in a byte, the even column in the low half
    codes = torch.randn((N, K), generator=g, device="cuda").mul_(2.7).round_().clamp_(-8, 7).add_(8).to(torch.uint8)
    codes = codes[:, 0::2] | (codes[:, 1::2] << 4)
    scales = ((torch.rand((N, -(-K // G)), generator=g, device="cuda") + 0.5) * 0.02).bfloat16()
    s = {"case": case, "codes": codes, "scales": scales}
    x = _activations((T, K), g)
    if case["act"] == "bf16":
        s["x"] = x.bfloat16()
    else:  # int8 rows with their group scales
        pad = -K % G
        a = torch.nn.functional.pad(x.abs(), (0, pad)).view(T, -1, G).amax(-1)
        xs = a / 127
        s["q"] = torch.round(x / xs.repeat_interleave(G, 1)[:, :K]).to(torch.int8)
        s["qs"] = xs
    return s


def _most_new(case):
    """The most new tokens of a request in a step of spans."""
    return min(256, case["chunk"] // 4)


def _plan_inputs(case, seed):
    g = _gen(seed, "cpu")
    B, C, ctx, L = case["batch"], case["chunk"], case["context"], case["layers"]
    pages = -(-ctx // PAGE)
    if case["kind"] == "decode":
        computed = torch.randint(ctx // 2, ctx, (B,), generator=g)
        new = torch.ones(B, dtype=torch.int64)
    else:
        # spans that end at or before the chunk's end; some start a chunk (its boundary commit falls to this step);
        # the step's buffers hold the most tokens that such a step may have, so some of them stay unused
        computed = torch.randint(0, ctx, (B,), generator=g)
        starts = torch.rand(B, generator=g) < 0.3
        computed = torch.where(starts, computed // C * C, computed)
        room = torch.minimum(C - computed % C, ctx - computed)
        most = _most_new(case)
        new = (1 + (torch.rand(B, generator=g) * most).long().clamp(max=most - 1)).minimum(room)
    slot = torch.randperm(B, generator=g)
    pad = case["padded"]
    if pad:  # rows that a captured batch has and this step does not use
        computed, new = (torch.cat((t, torch.zeros(pad, dtype=torch.int64))) for t in (computed, new))
        slot = torch.cat((slot, torch.full((pad,), -1)))
    table = torch.randperm(B * pages, generator=g).view(B, pages)
    ring_pages = 2 * C // PAGE
    src_pages = B * pages + 1
    base = src_pages + torch.arange(L) * (ring_pages * B + 1)
    tokens = slot.numel() if case["kind"] == "decode" else B * _most_new(case)

    def dev(t):
        return t.to(torch.int32).cuda()

    return {"case": case, "computed": dev(computed), "new": dev(new), "slot": dev(slot), "table": dev(table),
            "base": dev(base), "tokens": tokens, "max_tokens": ctx, "scratch_src": B * pages,
            "scratch_ring": ring_pages * B}


def prepare(case, seed):
    s = {"rows": _rows_inputs, "w4": _w4_inputs, "plan": _plan_inputs}[case["op"]](case, seed)
    if own:
        from lastkv_b200 import ops

        if case["op"] == "w4":  # the weight in the layout that a program loads it into, once
            s["weight"] = ops.w4_pack(s["codes"], s["scales"], case["group"])
            if case["act"] == "int8":
                s["rows"] = ops.Q8Rows(s["q"], s["qs"], case["group"])
        elif case["op"] == "plan":  # the step's static buffers
            B = s["slot"].numel()
            s["plan"] = ops.StepPlan(B, s["tokens"], s["table"], s["base"], chunk_size=case["chunk"],
                                     max_sequence_tokens=s["max_tokens"], scratch_src_page=s["scratch_src"],
                                     scratch_ring_page=s["scratch_ring"])
    return s


# ---------------------------------------------------------------- plain forms


def _groups(y, G):
    """[T, K] in groups of G columns, the last one filled up with zeros."""
    return torch.nn.functional.pad(y, (0, -y.shape[1] % G)).view(y.shape[0], -1, G)


def _rows_plain(s):
    c, x = s["case"], s["x"].float()
    out = {}
    if c["mode"] == "norm":
        h = x + s["residual"].float()
        out["h"] = h.bfloat16()
        y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + s["eps"]) * s["weight"].float()
    elif c["mode"] == "silu":
        gate, up = x[:, : c["cols"]], x[:, c["cols"]:]
        y = gate / (1 + torch.exp(-gate)) * up
    else:
        y = x
    y = _groups(y, c["group"])
    scale = y.abs().amax(-1) / 127
    q = torch.where(scale[..., None] == 0, 0, torch.round(y / scale[..., None]))
    out["scale"] = scale
    out["y"] = (q * scale[..., None]).view(x.shape[0], -1)[:, : c["cols"]].bfloat16()
    return out


def _w4_plain(s):
    c = s["case"]
    K, G = c["k"], c["group"]
    u = torch.stack((s["codes"] & 15, s["codes"] >> 4), -1).view(c["n"], K)
    w = (u.float() - 8) * s["scales"].float().repeat_interleave(G, 1)[:, :K]
    if c["act"] == "bf16":
        x = s["x"].float()
    else:
        x = s["q"].float() * s["qs"].repeat_interleave(G, 1)[:, :K]
    return (x @ w.T).bfloat16()


def _plan_plain(s):
    c = s["case"]
    C, L, T = c["chunk"], c["layers"], s["tokens"]
    p0, n, slot, table = s["computed"].long(), s["new"].long(), s["slot"].long(), s["table"].long()
    B, RP, W = slot.numel(), 2 * C // PAGE, table.shape[1] + 2 * C // PAGE
    dev = slot.device
    real = slot >= 0
    n = torch.where(real, n, 1)
    sl = slot.clamp(min=0)
    last = p0 + n - 1
    rec = (torch.div(last, C, rounding_mode="floor") * C - C).clamp(min=0)
    nsrc = torch.where(real, torch.div(rec, PAGE, rounding_mode="floor"), 0)
    npages = torch.div(last - rec + PAGE, PAGE, rounding_mode="floor")
    j = torch.arange(W, device=dev)[None]
    from_table = table[sl][:, torch.arange(W, device=dev).clamp(max=table.shape[1] - 1)]
    ring = sl[:, None] * RP + (nsrc[:, None] % RP + j - nsrc[:, None]) % RP
    bt = torch.where(j < nsrc[:, None], from_table, torch.where(j < (nsrc + npages)[:, None], ring, 0))
    bt = torch.where(real[:, None], bt, torch.where(j == 0, s["scratch_ring"], 0))
    bt_all = torch.where(j[None] < nsrc[None, :, None], bt[None], bt[None] + s["base"].long()[:, None, None])
    cu = torch.cat((n.new_zeros(1), n.cumsum(0)))
    tok = torch.arange(T, device=dev)
    row = torch.searchsorted(cu[1:], tok, right=True)  # B for the tokens that no row has
    ok = (row < B) & real[row.clamp(max=B - 1)]
    row = row.clamp(max=B - 1)
    pos = torch.where(ok, p0[row] + tok - cu[row], 0)
    src = table[sl[row], torch.div(pos, PAGE, rounding_mode="floor")] * PAGE + pos % PAGE
    commit = real & (p0 > 0) & (p0 % C == 0)
    order = torch.argsort(torch.where(commit, 0, 1), stable=True)
    count = commit.sum()
    page = torch.arange(C // PAGE, device=dev)[None]
    first = torch.div(p0[order] - C, PAGE, rounding_mode="floor").clamp(min=0)[:, None]
    live = (torch.arange(B, device=dev) < count)[:, None]
    raw = torch.where(live, table[sl[order][:, None], (first + page).clamp(max=table.shape[1] - 1)], 0)
    cring = torch.where(live, s["base"].long()[0] + sl[order][:, None] * RP + first % RP + page, 0)
    return {"block_tables": bt_all.int(), "seq_k": torch.where(real, last + 1, 1).int(), "cu_q": cu.int(),
            "positions": pos,
            "ring_slots": torch.where(ok, sl[row] * 2 * C + pos % (2 * C), s["scratch_ring"] * PAGE),
            "src_slots": torch.where(ok, src, s["scratch_src"] * PAGE),
            "commit_raw": raw.int(), "commit_ring": cring.int(), "commit_count": count.view(1).int()}


# ---------------------------------------------------------------- the framework's


def _rows_own(s):
    from lastkv_b200 import ops

    c, out = s["case"], {}
    if c["mode"] == "norm":
        out["h"], rows = ops.rmsnorm_q8(s["x"], s["weight"], s["eps"], s["residual"], group=c["group"])
    elif c["mode"] == "silu":
        rows = ops.silu_mul_q8(s["x"], group=c["group"])
    else:
        rows = ops.quantize_q8(s["x"], group=c["group"])
    out["scale"] = rows.scale
    out["y"] = ops.dequantize_q8(rows)  # the values that the 8 bits stand for
    return out


def _w4_own(s):
    from lastkv_b200 import ops

    return ops.w4_linear(s["x"] if s["case"]["act"] == "bf16" else s["rows"], s["weight"])


def _plan_own(s):
    p = s["plan"]
    p.run(s["computed"], s["new"], s["slot"])
    return {"block_tables": p.block_tables, "seq_k": p.seq_k, "cu_q": p.cu_q, "positions": p.positions,
            "ring_slots": p.ring_slots, "src_slots": p.src_slots, "commit_raw": p.commit_raw,
            "commit_ring": p.commit_ring, "commit_count": p.commit_count}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"rows": _rows_own, "w4": _w4_own, "plan": _plan_own}[op](state)
    return {"rows": _rows_plain, "w4": _w4_plain, "plan": _plan_plain}[op](state)


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    if case["op"] == "rows":
        T, H = case["rows"], case["cols"]
        per = {"norm": 2 + 2 + 2, "silu": 4, "plain": 2}[case["mode"]] + 1  # read, residual written, int8 written
        flops = {"norm": 10, "silu": 10, "plain": 4}[case["mode"]]
        # and the dequantised rows: int8 read, bf16 written
        return {"bytes": T * (H * (per + 3) + 2 * 4 * -(-H // case["group"])) + (2 * H if case["mode"] == "norm" else 0),
                "flops": flops * T * H}
    if case["op"] == "w4":
        T, N, K, G = case["tokens"], case["n"], case["k"], case["group"]
        g = -(-K // G)
        x = T * K * 2 if case["act"] == "bf16" else T * (K + 4 * g)
        return {"bytes": N * K // 2 + 2 * N * g + x + 2 * T * N, "flops": 2 * T * N * K}
    B, ctx, L = case["batch"] + case["padded"], case["context"], case["layers"]
    W = -(-ctx // PAGE) + 2 * case["chunk"] // PAGE
    tokens = B if case["kind"] == "decode" else B * _most_new(case)
    return {"bytes": 4 * B * W * L + 2 * B * W + 24 * tokens + 16 * B, "flops": B * W * L}


# ---------------------------------------------------------------- the definitions in 64 bits


def _exact_rows(s):
    c = s["case"]
    T, H, G = c["rows"], c["cols"], c["group"]
    x = s["x"].double()
    out = {}
    if c["mode"] == "norm":
        y = x.add(s["residual"].double())
        out["h"] = y.clone()
        y.div_((y.square().sum(1) / H + s["eps"]).sqrt()[:, None]).mul_(s["weight"].double())
    elif c["mode"] == "silu":
        y = x[:, :H].mul(torch.sigmoid(x[:, :H])).mul(x[:, H:])
    else:
        y = x
    n = -(-H // G)
    which = torch.arange(H, device=x.device) // G
    top = torch.zeros((T, n), dtype=torch.float64, device=x.device)
    top.scatter_reduce_(1, which.expand(T, H), y.abs(), "amax")
    step = (top / 127.0)[:, which]
    out["scale"] = top / 127.0
    out["y"] = torch.where(step > 0, torch.round(y / step) * step, torch.zeros_like(y))
    return out


def _exact_w4(s):
    c = s["case"]
    N, K, G = c["n"], c["k"], c["group"]
    col = torch.arange(K, device="cuda")
    w = torch.empty((N, K), dtype=torch.float64, device="cuda")
    w[:, 0::2] = (s["codes"].int() % 16 - 8).double()
    w[:, 1::2] = (s["codes"].int() // 16 - 8).double()
    w *= s["scales"].double()[:, col // G]
    if c["act"] == "bf16":
        x = s["x"].double()
    else:
        x = s["q"].double() * s["qs"].double()[:, col // G]
    return torch.einsum("tk,nk->tn", x, w)


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers only
    if case["op"] == "rows":
        return _exact_rows(_rows_inputs(case, seed))
    return _exact_w4(_w4_inputs(case, seed))
