"""Plain 64-bit forms of the decode-step operators, with error bounds for their 16-bit results.

A rounding to a type is off by at most half a step: HALF[dtype], relative to the value. fp32
roundings inside a kernel count 2^-24 each.
"""

import torch

HALF = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
F32 = 2.0**-24


def norm(x, weight, eps, residual=None):
    h = x.double() + (0 if residual is None else residual.double())
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * weight.double()
    return y, h


# Of a row's sum of squares each thread adds up at most 48 products (long rows: 1024 threads and
# rows up to 40000 in the tests), 10 more additions join them: 58 roundings of the sum, 29 of its
# root; the mean, eps, the reciprocal root (2 units) and two products are 8 more.
NORM_F32 = 40 * F32


def positions(table_row, n, page):
    at = torch.arange(n)
    return table_row.cpu().long()[at // page], at % page


def attention(q, k_cache, v_cache, table, lens, scale):
    """Outputs in 64 bits, their error bound for a kernel of 16-bit results, and the probabilities
    [hkv, group, n] of each sequence.

    The scores: products of 16-bit numbers are exact in fp32; a tensor core adds them 16 at a time,
    each addition off by at most 2^-22 of the sum of the products' absolute values (truncation), so
    a score is off by (dim / 16 + 2) 2^-22 scale sum|q k|, and scaling it, subtracting the maximum
    and taking 2^x add 4 2^-24 |s| and 2^-22. A probability is off by twice that (its own and the
    sum's), the product with v by 2^-16 more (the probability as a pair of 16-bit numbers), and the
    sums over n / 64 tiles of a warp, 4 warps and up to 512 blocks by (n / 64 + 520) 2^-23."""
    batch, hq, dim = q.shape
    page, hkv = k_cache.shape[1], k_cache.shape[2]
    group = hq // hkv
    out = torch.zeros(batch, hq, dim, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    probs, rel = [], []
    for b, n in enumerate(lens):
        if n == 0:
            probs.append(None)
            rel.append(0.0)
            continue
        pages, offs = positions(table[b], n, page)
        k = k_cache[pages, offs].double()
        v = v_cache[pages, offs].double()
        qb = q[b].double().view(hkv, group, dim)
        s = torch.einsum("hgd,nhd->hgn", qb, k) * scale
        size = torch.einsum("hgd,nhd->hgn", qb.abs(), k.abs()).max().item() * abs(scale)
        off = (dim / 16 + 2) * 2.0**-22 * size + 4 * F32 * s.abs().max().item() + 2.0**-22
        p = torch.softmax(s, -1)
        o = torch.einsum("hgn,nhd->hgd", p, v).reshape(hq, dim)
        spread = torch.einsum("hgn,nhd->hgd", p, v.abs()).reshape(hq, dim)
        out[b] = o
        bound[b] = HALF[q.dtype] * o.abs() + (2 * off + 2.0**-16 + (n / 64 + 520) * 2.0**-23) * spread
        # the smallest fp16 numbers have an absolute step
        bound[b] += 2.0**-25 if q.dtype == torch.float16 else 0.0
        probs.append(p)
        rel.append(2 * off + (n / 64 + 520) * 2.0**-23 + 2.0**-20)
    return out, bound, probs, rel


def evict(weights, table, lens, page, budget, recent):
    """kept [batch, hkv, budget] and the new lengths, in plain Python order: largest weight first (a
    NaN above all, -0 like 0), of equal ones the lowest position."""
    hkv = weights.shape[1]
    kept = torch.full((len(lens), hkv, budget), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        if n <= budget:
            kept[b, :, :n] = torch.arange(n, dtype=torch.int32)
            continue
        pages, offs = positions(table[b], n, page)
        for h in range(hkv):
            w = weights[pages, h, offs].double().cpu().tolist()
            old = n - recent
            ranked = sorted(range(old), key=lambda j: (w[j] == w[j], -w[j] if w[j] == w[j] else 0.0, j))
            chosen = sorted(ranked[:budget - recent]) + list(range(old, n))
            kept[b, h] = torch.tensor(chosen, dtype=torch.int32)
    return kept, torch.tensor([min(n, budget) for n in lens], dtype=torch.int32)


def logprobs(logits, tokens, top):
    """(logprobs, entropy, top logprobs, top ids) in 64 bits, and the bounds of the first two.

    The sum of e^(x - m): a thread adds up to vocab / 512 terms and 20 joins follow, each term is
    off by 2^-22 (2^x) and by |x - m| 2^-23 e^(x - m) <= 2^-24 of the largest: relative
    (vocab / 512 + 40) 2^-24 + 2^-21, the same for the sum of e^(x - m) (x - m), whose terms'
    absolute values add up to log vocab at most 16 here. The differences round at 2^-24 of what
    they are taken of."""
    x = logits.double()
    vocab = x.shape[1]
    # differences from the maximum: of values of 1e38, 64 bits do not hold x - lse either. A row with
    # a +inf, or with nothing above -inf, has no softmax: NaN, as inf - inf gives it
    top_x = x.amax(-1, keepdim=True)
    log_p = x - torch.where(top_x.isinf(), float("nan"), top_x)
    log_p = log_p - torch.log(torch.exp(log_p).sum(-1, keepdim=True))
    p = torch.exp(log_p)
    entropy = -torch.xlogy(p, p).sum(-1)
    ok = (tokens >= 0) & (tokens < vocab)
    lp = log_p.gather(1, tokens.clamp(0, vocab - 1)[:, None])[:, 0]
    lp = torch.where(ok, lp, float("nan"))
    ids = torch.sort(logits.float() + 0.0, dim=-1, descending=True, stable=True).indices[:, :top]
    off = (vocab / 512 + 40) * F32 + 2.0**-21
    finite = torch.where(torch.isfinite(x), x, 0.0)
    size = finite.amax(-1) - finite.amin(-1) + 20
    return (lp, entropy, log_p.gather(1, ids), ids), off + 4 * F32 * size, 2 * off * (size + 1)
