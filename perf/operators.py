"""The decode-step operators around the W4A16 GEMV, as cases to measure.

add_rms_norm (16- or 8-bit output), paged_attention, paged_evict and token_logprobs: the inputs a
serving loop has in hand, one pass through each operator (the plain form in torch operations, or
the package's kernels where `own` is true), the work a pass cannot do without, and the results in
64 bits.
"""

import functools
import math
import random
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
EPS = 1e-5
E4M3_MAX = 448.0
SCALE_FLOOR = 1e-12  # of the 8-bit scales, so that a row of zeros divides by something


@functools.lru_cache(maxsize=None)
def _ops():
    path = str(Path(__file__).resolve().parents[1] / "int4-gemv-cuda_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from int4gemv import ops

    return ops


# ---- cases ---------------------------------------------------------------------------------------


def _norm(rows, hidden, dtype, out, residual=True, **name):
    return dict(name, op="norm", rows=rows, hidden=hidden, dtype=dtype, out=out, residual=residual)


def _attn(batch, longest, hq, hkv, dim, page, dtype, append, adds, lens=1, **name):
    """append: the call writes the new token's k and v; adds: it adds up the attention weights."""
    return dict(name, op="attn", batch=batch, longest=longest, hq=hq, hkv=hkv, dim=dim, page=page,
                dtype=dtype, append=append, adds=adds, lens=lens)


def _evict(batch, longest, hkv, dim, page, dtype, budget, recent, lens=1, **name):
    return dict(name, op="evict", batch=batch, longest=longest, hkv=hkv, dim=dim, page=page,
                dtype=dtype, budget=budget, recent=recent, lens=lens)


def _logprobs(rows, vocab, dtype, top, masked=False, **name):
    return dict(name, op="logprobs", rows=rows, vocab=vocab, dtype=dtype, top=top, masked=masked)


def listed():
    return [
        # the norm before a projection in a decode step of one sequence: latency
        _norm(1, 4096, "fp16", "same", name="norm 1x4096"),
        # a decode batch of odd size
        _norm(37, 8192, "bf16", "same", name="norm 37x8192"),
        # a prompt batch whose next product takes 8-bit activations
        _norm(6000, 8192, "fp16", "e4m3", name="norm 6000x8192 e4m3"),
        # one chat turn's decode step (q 4096 rows, k and v 1024, the grouped launch's sizes): latency
        _attn(1, 701, 32, 8, 128, 16, "fp16", True, False, name="attn 1x701"),
        # a decode batch of uneven lengths that also adds up the weights eviction goes by
        _attn(24, 4096, 32, 8, 128, 16, "bf16", True, True, name="attn 24x4096 weights"),
        # one long document: few rows, the cache's length split over the whole card
        _attn(1, 131072, 64, 8, 128, 64, "fp16", False, False, name="attn 1x131072"),
        # a full serving batch (8192 hidden: 64 query heads), uneven lengths
        _attn(64, 8192, 64, 8, 128, 32, "fp16", True, False, name="attn 64x8192"),
        # one sequence over its budget: latency of the choice
        _evict(1, 2503, 8, 128, 16, "fp16", 1001, 203, name="evict 1x2503"),
        # a batch shrunk to a quarter at once
        _evict(32, 8192, 8, 128, 32, "bf16", 2048, 512, name="evict 32x8192"),
        # one sampled token with its alternatives, a 32000-word vocabulary and one added word
        _logprobs(1, 32001, "fp16", 5, name="logprobs 1x32001"),
        # a full decode batch of the GEMV, grammar-masked logits, the most alternatives usually asked
        _logprobs(64, 128256, "fp16", 20, masked=True, name="logprobs 64x128256"),
        # scoring a prompt, a few alternatives a token
        _logprobs(2048, 128256, "bf16", 3, name="logprobs 2048x128256"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "attn", "attn", "evict", "logprobs"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "norm":
        hidden = rng.choice([_log_int(rng, 64, 16384), 8 * _log_int(rng, 16, 2048)])
        rows = _log_int(rng, 1, max(1, min(16384, 6000 * 8192 // hidden)))
        dtype = rng.choice(["fp16", "bf16", "fp32"])
        return _norm(rows, hidden, dtype, rng.choice(["same", "e4m3"]), rng.random() < 0.75)
    if op == "attn":
        hkv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16])
        dim = rng.choice([64, 80, 96, 128, 192, 256])
        batch = _log_int(rng, 1, 64)
        most = max(64, min(131072, 64 * 8192 * 8 * 128 // ((batch + 1) * hkv * dim)))
        return _attn(batch, _log_int(rng, 16, most), group * hkv, hkv, dim,
                     rng.choice([8, 16, 32, 48, 64, 128, 256]), dtype, rng.random() < 0.6,
                     rng.random() < 0.5, rng.randrange(1 << 20))
    if op == "evict":
        hkv, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 128, 256])
        batch = _log_int(rng, 1, 32)
        most = max(64, min(65536, 32 * 8192 * 8 * 128 // (batch * hkv * dim)))
        longest = _log_int(rng, 32, most)
        budget = max(1, min(int(longest * rng.uniform(0.15, 0.8)), 32 * 2048 * 8 * 128 // (batch * hkv * dim)))
        return _evict(batch, longest, hkv, dim, rng.choice([8, 16, 32, 48, 64, 128]), dtype, budget,
                      int(budget * rng.uniform(0.0, 0.6)), rng.randrange(1 << 20))
    vocab = _log_int(rng, 1000, 262144)
    dtype = rng.choice(["fp16", "bf16", "fp32"])
    rows = _log_int(rng, 1, max(1, 2048 * 128256 // (2 * vocab)))
    return _logprobs(min(rows, 4096), vocab, dtype, rng.choice([0, 1, 3, 5, 8, 20, 32]), rng.random() < 0.3)


def _lengths(case):
    """Uneven lengths up to `longest`: one sequence is the longest, and of a batch of eight or more
    one slot is empty (padding of a captured batch)."""
    r = random.Random(case["lens"])
    low = max(1, case["longest"] // 16)
    lens = [r.randint(low, case["longest"]) for _ in range(case["batch"])]
    lens[r.randrange(len(lens))] = case["longest"]
    if len(lens) >= 8:
        lens[lens.index(case["longest"]) - 1] = 0
    return lens


# ---- inputs --------------------------------------------------------------------------------------


def _pages(lens, page, width, first, order):
    """A block table [B, width] of pages from `order` (a permutation), -1 where none is needed."""
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = first
    for b, n in enumerate(lens):
        need = -(-n // page)
        table[b, :need] = order[at:at + need]
        at += need
    return table, at


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dtype):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)

    s = dict(case)
    if case["op"] == "norm":
        t, h = case["rows"], case["hidden"]
        s["x"] = normal(t, h)
        # a residual stream: wider than what is added to it, a few channels far out
        s["r"] = normal(t, h, std=4.0) if case["residual"] else None
        if case["residual"]:
            s["r"][:, :: max(1, h // 7)] *= 8
        s["w"] = (1 + 0.2 * torch.randn(h, generator=g, device="cuda")).to(dtype)
        return s
    if case["op"] == "logprobs":
        t, v = case["rows"], case["vocab"]
        s["logits"] = normal(t, v, std=2.5)
        peak = torch.randint(v, (t, 12), generator=g, device="cuda")
        rise = 14 * torch.rand(t, 12, generator=g, device="cuda")
        s["logits"].scatter_(1, peak, rise.to(dtype))
        s["tokens"] = peak[:, 0].contiguous()  # mostly likely tokens
        if case["masked"]:  # a grammar leaves every third word or so
            keep = torch.rand(v, generator=g, device="cuda") < 0.3
            keep[:32] = True
            s["logits"].masked_fill_(~keep, float("-inf"))
        return s
    lens, page, hkv, dim = _lengths(case), case["page"], case["hkv"], case["dim"]
    width = -(-case["longest"] // page)
    used = sum(-(-n // page) for n in lens)
    budget = case.get("budget", 0)
    new_lens = [min(n, budget) for n in lens]
    total = used + (sum(-(-n // page) for n in new_lens) if budget else 0) + 3
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table, at = _pages(lens, page, width, 0, order)
    s["table"] = table.cuda()
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["longest_page"] = width
    s["k_cache"] = normal(total, page, hkv, dim)
    s["v_cache"] = normal(total, page, hkv, dim)
    # weights as they add up over decode steps: most positions little, some a lot
    s["weights"] = torch.rand(total, hkv, page, generator=g, device="cuda").pow_(8).mul_(20)
    if case["op"] == "evict":
        s["new_table"] = _pages(new_lens, page, -(-budget // page), at, order)[0].cuda()
        return s
    b = case["batch"]
    s["q"] = normal(b, case["hq"], dim, std=1.5)
    s["scale"] = 1.0 / math.sqrt(dim)
    s["k"] = normal(b, hkv, dim) if case["append"] else None
    s["v"] = normal(b, hkv, dim) if case["append"] else None
    # an empty slot of the plain form's batched write rewrites a place here that no table names
    s["spare"] = int(order[-1])
    return s


# ---- one pass ------------------------------------------------------------------------------------


def run(s):
    return {"norm": _run_norm, "attn": _run_attn, "evict": _run_evict, "logprobs": _run_logprobs}[s["op"]](s)


def _run_norm(s):
    if own:
        if s["out"] == "same":
            return _ops().add_rms_norm(s["x"], s["w"], EPS, s["r"])
        return _ops().add_rms_norm_quant(s["x"], s["w"], EPS, s["r"])
    h = s["x"].float() + s["r"].float() if s["r"] is not None else s["x"].float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["w"].float()
    h = h.to(s["x"].dtype)
    if s["out"] == "same":
        return y.to(s["x"].dtype), h
    scales = (y.abs().amax(-1) / E4M3_MAX).clamp_min(SCALE_FLOOR)
    return (y / scales[:, None]).to(torch.float8_e4m3fn), scales, h


def _run_attn(s):
    w = s["weights"] if s["adds"] else None
    if own:
        out = _ops().paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"],
                                     s["scale"], s["k"], s["v"], w)
    else:
        b, hq, dim = s["q"].shape
        hkv, page = s["hkv"], s["page"]
        n = s["lens"].long()
        pos = torch.arange(s["longest_page"] * page, device="cuda")
        valid = pos < n[:, None]  # [B, L]
        pages = s["table"].long().clamp_min(0)
        if s["k"] is not None:
            some = n > 0
            last = (n - 1).clamp_min(0)
            at = torch.where(some, pages.gather(1, (last // page)[:, None])[:, 0], s["spare"])
            off = last % page
            for cache, new in ((s["k_cache"], s["k"]), (s["v_cache"], s["v"])):
                cache[at, off] = torch.where(some[:, None, None], new, cache[at, off])
            if w is not None:
                w[at, :, off] = torch.where(some[:, None], 0.0, w[at, :, off])
        keys = s["k_cache"][pages].float().view(b, -1, hkv, dim)
        values = s["v_cache"][pages].float().view(b, -1, hkv, dim)
        values = values.masked_fill_(~valid[:, :, None, None], 0.0)
        qf = s["q"].float().view(b, hkv, hq // hkv, dim)
        scores = torch.einsum("bhgd,blhd->bhgl", qf, keys) * s["scale"]
        scores = scores.masked_fill_(~valid[:, None, None, :], float("-inf"))
        top = scores.amax(-1, keepdim=True).clamp_min(-3e38)  # of an empty row: anything finite
        e = torch.exp(scores - top)
        p = e / e.sum(-1, keepdim=True).clamp_min(1e-38)
        out = torch.einsum("bhgl,blhd->bhgd", p, values).reshape(b, hq, dim).to(s["q"].dtype)
        if w is not None:
            # behind a sequence's end zeros are added
            where = pages.repeat_interleave(page, 1), (pos % page).expand(b, -1)
            w.permute(0, 2, 1).index_put_(where, p.sum(2).permute(0, 2, 1), accumulate=True)
    got = [out]
    if s["k"] is not None:
        got += [s["k_cache"], s["v_cache"]]
    return got + ([w] if w is not None else [])


def _run_evict(s):
    if own:
        kept, lens = _ops().paged_evict(s["k_cache"], s["v_cache"], s["weights"], s["table"],
                                        s["lens"], s["new_table"], s["budget"], s["recent"])
    else:
        b, hkv, page, budget, recent = s["batch"], s["hkv"], s["page"], s["budget"], s["recent"]
        n = s["lens"].long()[:, None, None]
        pages = s["table"].long().clamp_min(0)
        w = s["weights"][pages].transpose(1, 2).reshape(b, hkv, -1)  # [B, H, L]
        pos = torch.arange(w.shape[-1], device="cuda")
        # what is always kept first, what is not there last; of the rest the largest weight
        w = torch.where(pos >= n - recent, float("inf"), w)
        w = torch.where(pos < n, w, float("-inf"))
        best = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :budget]
        best = best.where(torch.arange(best.shape[-1], device="cuda") < n, w.shape[-1])
        kept = torch.sort(best, dim=-1).values  # [B, H, budget], in order, absent ones last
        lens = n[:, 0, 0].clamp_max(budget)
        j = torch.arange(kept.shape[-1], device="cuda")
        here = j < lens[:, None]  # [B, budget], the same for every head
        bi, ji = here.nonzero(as_tuple=True)
        src = kept.transpose(1, 2)[bi, ji]  # [N, H]
        heads = torch.arange(hkv, device="cuda")
        page_from, off_from = pages[bi[:, None], src // page], src % page
        page_to, off_to = s["new_table"].long()[bi, ji // page][:, None], (ji % page)[:, None]
        for cache in (s["k_cache"], s["v_cache"]):
            cache[page_to, off_to, heads] = cache[page_from, off_from, heads]
        s["weights"][page_to, heads, off_to] = s["weights"][page_from, heads, off_from]
        kept = torch.where(here[:, None, :], kept, -1).to(torch.int32)
        lens = lens.to(torch.int32)
    return [kept, lens, s["k_cache"], s["v_cache"], s["weights"]]


def _run_logprobs(s):
    if own:
        return _ops().token_logprobs(s["logits"], s["tokens"], s["top"])
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    z = e.sum(-1, keepdim=True, dtype=torch.float64)
    log_z = torch.log(z)
    logprobs = (x.gather(1, s["tokens"][:, None]) - top - log_z)[:, 0].float()
    entropy = (log_z - torch.where(e > 0, e * (x - top), 0.0).sum(-1, keepdim=True, dtype=torch.float64) / z)[:, 0].float()
    if s["top"]:
        best = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :s["top"]].contiguous()
    else:
        best = s["tokens"].new_empty((x.shape[0], 0))
    return logprobs, entropy, (x.gather(1, best) - top - log_z).float(), best


# ---- what a pass cannot do without -----------------------------------------------------------------


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "norm":
        n = case["rows"] * case["hidden"]
        read = n * e * (2 if case["residual"] else 1) + case["hidden"] * e
        # without a residual the sum is x itself
        wrote = (n * e if case["residual"] else 0) + (n * e if case["out"] == "same" else n + 4 * case["rows"])
        return {"bytes": read + wrote, "flops": 6 * n}
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * e + case["rows"] * (16 + 12 * case["top"]), "flops": 5 * n}
    lens, hkv, dim = _lengths(case), case["hkv"], case["dim"]
    tokens = sum(lens)
    tables = 4 * sum(-(-n // case["page"]) for n in lens) + 4 * len(lens)
    if case["op"] == "evict":
        kept = sum(min(n, case["budget"]) for n in lens)
        row = hkv * (2 * dim * e + 4)
        return {"bytes": 4 * tokens * hkv + 2 * kept * row + tables + 4 * len(lens) * (hkv * case["budget"] + 1),
                "flops": tokens * hkv}
    row = hkv * 2 * dim * e
    some = sum(1 for n in lens if n)
    moved = tokens * row + 2 * len(lens) * case["hq"] * dim * e + tables
    if case["append"]:
        moved += some * row  # its k and v are read from the call's, and written
    if case["adds"]:
        moved += 8 * tokens * hkv
    return {"bytes": moved, "flops": 4 * case["hq"] * dim * tokens}


# ---- the results in 64 bits ------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double()
        if s["r"] is not None:
            h = h + s["r"].double()
        y = h / torch.sqrt((h * h).sum(-1, keepdim=True) / h.shape[1] + EPS) * s["w"].double()
        if case["out"] == "same":
            return y, h
        scales = torch.clamp(y.abs().max(-1).values / E4M3_MAX, min=SCALE_FLOOR)
        return y / scales[:, None], scales, h  # like the 16-bit outputs, before their rounding
    if case["op"] == "logprobs":
        parts = []
        for i in range(0, case["rows"], 256):
            x = s["logits"][i:i + 256].double()
            t = s["tokens"][i:i + 256]
            lse = torch.logsumexp(x, -1)
            p = torch.exp(x - lse[:, None])
            entropy = -torch.xlogy(p, p).sum(-1)
            # the order of the values, then of the places: one key for both
            ids = torch.argsort(x, dim=-1, descending=True, stable=True)[:, :case["top"]]
            rows = torch.arange(x.shape[0], device="cuda")
            parts.append((x[rows, t] - lse, entropy, torch.take_along_dim(x, ids, 1) - lse[:, None], ids.contiguous()))
        return tuple(torch.cat(c) for c in zip(*parts))
    lens, page, hkv, dim = _lengths(case), case["page"], case["hkv"], case["dim"]
    table = s["table"].cpu().long()
    if case["op"] == "evict":
        kept = torch.full((len(lens), hkv, case["budget"]), -1, dtype=torch.int32)
        new_table = s["new_table"].cpu().long()
        for b, n in enumerate(lens):
            m = min(n, case["budget"])
            if not m:
                continue
            at = torch.arange(n)
            rows, offs = table[b, at // page].cuda(), (at % page).cuda()
            to = torch.arange(m)
            rows_to, offs_to = new_table[b, to // page].cuda(), (to % page).cuda()
            for h in range(hkv):
                w = s["weights"][rows, h, offs].double().cpu()
                old = n - min(case["recent"], n)
                ranked = torch.argsort(-w[:old], stable=True).tolist()
                chosen = sorted(ranked[:m - (n - old)] + list(range(old, n)))
                kept[b, h, :m] = torch.tensor(chosen, dtype=torch.int32)
                pick = torch.tensor(chosen, device="cuda")
                for cache in (s["k_cache"], s["v_cache"]):
                    cache[rows_to, offs_to, h] = cache[rows[pick], offs[pick], h]
                s["weights"][rows_to, h, offs_to] = s["weights"][rows[pick], h, offs[pick]]
        new_lens = torch.tensor([min(n, case["budget"]) for n in lens], dtype=torch.int32)
        return [kept, new_lens, s["k_cache"], s["v_cache"], s["weights"].double()]
    out = torch.zeros(case["batch"], case["hq"], dim, dtype=torch.float64, device="cuda")
    weights = s["weights"].double()
    group = case["hq"] // hkv
    for b, n in enumerate(lens):
        if not n:
            continue
        at = torch.arange(n)
        rows, offs = table[b, at // page].cuda(), (at % page).cuda()
        if case["append"]:
            s["k_cache"][rows[-1], offs[-1]] = s["k"][b]
            s["v_cache"][rows[-1], offs[-1]] = s["v"][b]
            weights[rows[-1], :, offs[-1]] = 0
        for h in range(hkv):
            k, v = s["k_cache"][rows, offs, h].double(), s["v_cache"][rows, offs, h].double()
            p = torch.softmax(s["q"][b, h * group:(h + 1) * group].double() @ k.T * s["scale"], -1)
            out[b, h * group:(h + 1) * group] = p @ v
            weights[rows, h, offs] += p.sum(0)
    got = [out]
    if case["append"]:
        got += [s["k_cache"], s["v_cache"]]
    return got + ([weights] if case["adds"] else [])
