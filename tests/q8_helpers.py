"""Plain 64-bit forms of the 8-bit pages' operators and their error bounds."""

import torch

BF16_HALF_STEP = torch.finfo(torch.bfloat16).eps / 2  # 2^-8
FP32_HALF_STEP = torch.finfo(torch.float32).eps / 2   # 2^-24


def quantized(x):
    """Codes and scales (fp32 [pages, 2, Hkv]) of bf16 pages, by the formula; zeros where a block is not finite."""
    n, _, h, d = x.shape
    y = x.float().view(n, 2, 8, h, d)
    amax = y.abs().amax((2, 4))
    amax = torch.where(y.isnan().any(4).any(2), torch.nan, amax)
    scale = (amax.double() / 127).float()  # (a division by a number in fp32 is a product with its reciprocal in torch)
    s = scale[:, :, None, :, None].double()
    codes = torch.where((s == 0) | ~s.isfinite(), 0, torch.round(y.double() / s))
    return codes.view(x.shape), scale


def values(codes, scale):
    """What codes stand for, float64."""
    return codes.double() * scale.double().repeat_interleave(8, 1)[..., None]


def random_cache(seed, lens, num_q8, hkv, d, *, extra=5, spread=1.0, device="cuda"):
    """Shuffled tables over 8-bit and bf16 pages.  Returns a dict of device tensors with the 8-bit codes in natural order."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    B = len(lens)
    pages = [-(-n // 16) for n in lens]
    q8 = [min(a, b) for a, b in zip(num_q8, pages)]
    W = max(1, max(pages))
    n8, nb = sum(q8) + extra, sum(pages) - sum(q8) + extra
    p8, pb = torch.randperm(n8, generator=g), torch.randperm(nb, generator=g)
    table = torch.zeros((B, W), dtype=torch.int32)
    a = c = 0
    for b in range(B):
        table[b, :q8[b]] = p8[a:a + q8[b]]
        table[b, q8[b]:pages[b]] = pb[c:c + pages[b] - q8[b]]
        a, c = a + q8[b], c + pages[b] - q8[b]

    def codes():
        return torch.randint(-127, 128, (n8, 16, hkv, d), generator=g).to(torch.int8)

    def scales():
        return torch.exp(torch.randn((n8, 2, hkv), generator=g) * 0.5) * 0.015 * spread

    t = {"k": codes(), "v": codes(), "ks": scales(), "vs": scales(), "table": table,
         "num_q8": torch.tensor(num_q8, dtype=torch.int32), "seq_k": torch.tensor(lens, dtype=torch.int32),
         "pool_k": torch.randn((nb, 16, hkv, d), generator=g).bfloat16(),
         "pool_v": torch.randn((nb, 16, hkv, d), generator=g).bfloat16()}
    return {name: x.to(device) for name, x in t.items()}


def row_keys(t, b):
    """(K, V) float64 [n, Hkv, D] of row b."""
    n = int(t["seq_k"][b])
    pages = min(-(-n // 16), t["table"].shape[1])
    m = min(int(t["num_q8"][b]), pages)
    ids = t["table"][b].long()
    out = []
    for name in ("k", "v"):
        old = values(t[name][ids[:m]], t[name + "s"][ids[:m]])
        new = t["pool_" + name][ids[m:pages]].double()
        out.append(torch.cat((old, new)).flatten(0, 1)[:n])
    return out


def attention(q, k, v, scale, causal_from=None, weight_error=0.0):
    """One row's attention in 64 bits: q [L, Hq, D], k and v [n, Hkv, D].  Query i sees the keys up to
    causal_from + i (None: all).  Returns (out, bound): how far a kernel may be that sums in fp32, rounds each
    weight once to bf16 and the output once to bf16:
      - the output's rounding, half a step of |out|;
      - the weights', half a step each: half a step of sum p |v|;
      - a score is a sum of D products whose rounding moves it by at most e = D half steps (fp32) of
        scale * sum |q k|, twice that for the scaling, which changes a weight by a factor of exp(2 e) either way
        (once in the weight, once in the sum); the exponential's own error is `weight_error`;
      - sums of n weights and n products in fp32: n half steps each."""
    L, Hq, D = q.shape
    n, Hkv, _ = k.shape
    out = torch.zeros((L, Hq, D), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    if n == 0:
        return out, bound
    G = Hq // Hkv
    q, k, v = q.double(), k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = torch.einsum("lhd,nhd->lhn", q, k) * scale
    e = 2 * D * FP32_HALF_STEP * scale * torch.einsum("lhd,nhd->lhn", q.abs(), k.abs()).amax(-1, keepdim=True)
    if causal_from is not None:
        late = torch.arange(n, device=q.device)[None] > causal_from + torch.arange(L, device=q.device)[:, None]
        s = s.masked_fill(late[:, None], float("-inf"))
    some = (s > float("-inf")).any(-1, keepdim=True)
    p = torch.where(some, torch.softmax(s, -1), torch.zeros_like(s))
    out = torch.einsum("lhn,nhd->lhd", p, v)
    size = torch.einsum("lhn,nhd->lhd", p, v.abs())
    weights = BF16_HALF_STEP + torch.expm1(2 * e) + 2 * weight_error + 2 * n * FP32_HALF_STEP
    return out, BF16_HALF_STEP * out.abs() + (1 + BF16_HALF_STEP) * weights * size


def assert_within(got, ref, bound, what=""):
    off = (got.double() - ref).abs()
    over = off > bound + 1e-30
    assert not bool((over | ~torch.isfinite(got.double())).any()), \
        f"{what}: {int(over.sum())} values off, the worst by {float((off / (bound + 1e-30)).max()):.2f} bounds"
