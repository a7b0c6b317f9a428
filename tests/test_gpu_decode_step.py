"""The decode step as a user runs it: norm, grouped q / k / v, attention over the paged cache, output
projection with the residual, norm, gate / up, down projection, last norm, vocabulary projection,
log probabilities, and eviction when the cache is full. Every operator's output is checked against
its plain 64-bit form on the inputs it was given, so that each is held to its own bound."""

import math

import pytest
import torch

import decode_reference as ref
from int4gemv import capi, ops, quant, reference

pytestmark = pytest.mark.gpu

F16 = torch.float16
HIDDEN, HEADS, KV_HEADS, DIM, INNER, VOCAB, LAYERS, PAGE = 1024, 8, 2, 128, 1024, 2000, 2, 16
EPS, GROUP = 1e-5, 128


def packed(n, k, gen):
    return quant.quantize(torch.randn(n, k, generator=gen, device="cuda") * 0.03, GROUP)


class Model:
    def __init__(self, batch, lens, pages, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        sizes = [HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM]
        norm = lambda: (1 + 0.1 * torch.randn(HIDDEN, generator=g, device="cuda")).to(F16)  # noqa: E731
        self.qkv_sizes = sizes
        self.layers = []
        for _ in range(LAYERS):
            gate, up = packed(INNER, HIDDEN, g), packed(INNER, HIDDEN, g)
            self.layers.append(dict(
                n1=norm(), n2=norm(), qkv=packed(sum(sizes), HIDDEN, g), o=packed(HIDDEN, HEADS * DIM, g),
                gate_up=tuple(quant.interleave_rows(a, b) for a, b in zip(gate, up)),
                down=packed(HIDDEN, INNER, g),
                k=torch.randn(pages, PAGE, KV_HEADS, DIM, generator=g, device="cuda").to(F16),
                v=torch.randn(pages, PAGE, KV_HEADS, DIM, generator=g, device="cuda").to(F16),
                w=torch.rand(pages, KV_HEADS, PAGE, generator=g, device="cuda")))
        self.last_norm, self.head = norm(), packed(VOCAB, HIDDEN, g)
        self.x = torch.randn(batch, HIDDEN, generator=g, device="cuda").to(F16)
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        width = 8
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:batch * width]
        self.table = order.int().view(batch, width).cuda()

    def step(self, check=None):
        """One token a sequence; check(name, outputs, inputs) sees every operator's."""
        check = check or (lambda *a: None)
        scale = 1 / math.sqrt(DIM)
        x, h = self.x, None
        for layer in self.layers:
            before = x, h
            y, h = ops.add_rms_norm(x, layer["n1"], EPS, h)
            check("norm", (y, h), (*before, layer["n1"]))
            q, k, v = ops.w4a16_grouped(y, *layer["qkv"], GROUP, self.qkv_sizes)
            check("gemv", torch.cat([q, k, v], 1), (y, layer["qkv"]))
            q, k, v = (t.view(t.shape[0], -1, DIM) for t in (q, k, v))
            w_before = layer["w"].clone()
            a = ops.paged_attention(q, layer["k"], layer["v"], self.table, self.lens, scale, k, v, layer["w"])
            check("attention", (a, w_before, layer["w"]), (q, k, v, layer["k"], layer["v"], scale))
            a = a.view(a.shape[0], -1)
            h2 = ops.w4a16_bias_residual(a, *layer["o"], GROUP, residual=h)
            check("gemv", h2, (a, layer["o"], h))
            y, _ = ops.add_rms_norm(h2, layer["n2"], EPS)
            check("norm", (y, h2), (h2, None, layer["n2"]))
            inner = ops.w4a16_silu_mul(y, *layer["gate_up"], GROUP)
            check("silu", inner, (y, layer["gate_up"]))
            x, h = ops.w4a16(inner, *layer["down"], GROUP), h2
            check("gemv", x, (inner, layer["down"]))
        y, _ = ops.add_rms_norm(x, self.last_norm, EPS, h)
        logits = ops.w4a16(y, *self.head, GROUP)
        tokens = logits.argmax(-1)
        out = ops.token_logprobs(logits, tokens, 8)
        check("logprobs", out, (logits, tokens))
        return [y, logits, *out]


def checker(model):
    def within(got, want, bound, what):
        assert ((got.double() - want).abs() <= bound).all(), what

    def check(name, out, given):
        if name == "norm":
            x, r, w = given
            y, h = ref.norm(x, w, EPS, r)
            within(out[0], y, y.abs() * (ref.HALF[F16] + ref.NORM_F32) + 2.0**-25, "y")
            within(out[1], h, h.abs() * (ref.HALF[F16] + ref.F32) + 2.0**-25, "h")
        elif name == "gemv":
            want = given[0].float() @ quant.dequantize(*given[1], GROUP).T
            reference.assert_matches_reference(out, want + (given[2].float() if len(given) > 2 else 0))
        elif name == "silu":
            both = given[0].float() @ quant.dequantize(*given[1], GROUP).T
            reference.assert_matches_reference(out, torch.nn.functional.silu(both[:, ::2]) * both[:, 1::2])
        elif name == "attention":
            a, w_before, w_after = out
            q, k, v, kc, vc, scale = given
            lens = model.lens.tolist()
            want, bound, probs, rel = ref.attention(q, kc, vc, model.table, lens, scale)
            within(a, want, bound, "attention")
            total = w_before.double()
            off = torch.zeros_like(total)
            for b, n in enumerate(lens):
                if not n:
                    continue
                pages, offs = ref.positions(model.table[b], n, PAGE)
                assert torch.equal(kc[pages[-1], offs[-1]], k[b]) and torch.equal(vc[pages[-1], offs[-1]], v[b])
                p = probs[b].sum(1).T
                total[pages[-1], :, offs[-1]] = 0
                total[pages, :, offs] += p
                off[pages, :, offs] += p * (rel[b] + 4 * ref.F32)
            within(w_after, total, off + total * 2 * ref.F32, "weights")
        else:
            (lp, ent, top_lp, ids), off, off_ent = ref.logprobs(given[0], given[1], 8)
            assert torch.equal(out[3], ids)
            within(out[0], lp, off, "logprobs")
            within(out[1], ent, off_ent, "entropy")
            within(out[2], top_lp, off[:, None], "top")

    return check


@pytest.mark.parametrize("lens", [[100], [17, 0, 100, 64], [90] * 12])
def test_steps_with_eviction(lens):
    """Three steps, an eviction of the full sequences into new pages, and two more steps."""
    batch = len(lens)
    model = Model(batch, lens, pages=batch * 8 + batch * 4 + 2)
    used = set(model.table.flatten().tolist())
    spare = [p for p in range(batch * 12 + 2) if p not in used]
    grown = torch.tensor([int(n > 0) for n in lens], dtype=torch.int32, device="cuda")
    for step in range(5):
        model.lens += grown
        model.step(checker(model))
        if step == 2:
            new = torch.tensor(spare[:batch * 4], dtype=torch.int32, device="cuda").view(batch, 4)
            for layer in model.layers:
                old = layer["k"].clone(), layer["v"].clone(), layer["w"].clone()
                kept, new_lens = ops.paged_evict(layer["k"], layer["v"], layer["w"], model.table, model.lens,
                                                 new, 50, 20)
                want, want_lens = ref.evict(old[2], model.table, model.lens.tolist(), PAGE, 50, 20)
                assert torch.equal(kept.cpu(), want) and torch.equal(new_lens.cpu(), want_lens)
                for b, n in enumerate(want_lens.tolist()):
                    to_p, to_o = ref.positions(new[b], n, PAGE)
                    for h in range(KV_HEADS):
                        src = want[b, h, :n].long()
                        from_p, from_o = model.table[b].cpu().long()[src // PAGE], src % PAGE
                        assert torch.equal(layer["k"][to_p, to_o, h], old[0][from_p, from_o, h])
                        assert torch.equal(layer["v"][to_p, to_o, h], old[1][from_p, from_o, h])
                        assert torch.equal(layer["w"][to_p, h, to_o], old[2][from_p, h, from_o])
            model.table[:, :4] = new  # the fourth page has room for what follows
            model.lens.copy_(new_lens)
    assert capi.device_status() == 0


def test_step_in_a_captured_graph():
    """A whole step captured once gives the eager step's bits on every replay."""
    model = Model(2, [70, 33], pages=20, seed=3)
    state = [[layer[k].clone() for k in "kvw"] for layer in model.layers]

    def restore():
        for layer, was in zip(model.layers, state):
            for k, t in zip("kvw", was):
                layer[k].copy_(t)

    want = [t.clone() for t in model.step()]
    after = [[layer[k].clone() for k in "kvw"] for layer in model.layers]
    restore()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model.step()
    for _ in range(3):
        restore()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
        for layer, was in zip(model.layers, after):
            assert all(torch.equal(layer[k], t) for k, t in zip("kvw", was))
