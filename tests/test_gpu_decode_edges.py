"""The decode-step operators where they can go wrong: rows shorter than a chunk and more rows than a
grid has blocks, a tensor given twice, pages that are all refused, scores far apart."""

import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import decode_reference as ref
from int4gemv import capi, ops
from test_gpu_decode_ops import (BF16, F16, F32, Paged, assert_within, check_attention,  # noqa: F401
                                 check_evict, check_logprobs, gen, no_status_left, randn, same_bits)

pytestmark = pytest.mark.gpu


def check_norm(x, w, residual, eps=1e-5):
    """Both outputs of both forms against the 64-bit ones (the bounds of test_norm)."""
    dtype, rows, hidden = x.dtype, *x.shape
    want, h64 = ref.norm(x, w, eps, residual)
    y, h = ops.add_rms_norm(x, w, eps, residual)
    tiny = 2.0**-25 if dtype == F16 else 0.0
    assert_within(y, want, want.abs() * (ref.HALF[dtype] + ref.NORM_F32) + tiny, "y")
    assert_within(h, h64, h64.abs() * (ref.HALF[dtype] + ref.F32) + tiny, "h")
    q, scales, h2 = ops.add_rms_norm_quant(x, w, eps, residual)
    assert same_bits(h, h2)
    s64 = want.abs().amax(-1) / 448
    assert_within(scales, s64, s64 * (ref.NORM_F32 + 4 * ref.F32), "scales")
    v = want / s64[:, None]
    assert_within(q.float(), v, v.abs() * (2.0**-4 + 2 * ref.NORM_F32) + 2.0**-10, "q")


@pytest.mark.parametrize("rows,hidden,dtype", [
    (2, 1, F16), (10, 1, BF16), (3, 2, F16), (2, 3, F16), (7, 3, BF16), (2, 5, F16), (9, 6, BF16),
    (2, 1, F32), (5, 2, F32), (3, 3, F32)])
def test_norm_of_rows_shorter_than_a_chunk(rows, hidden, dtype):
    """Several rows in 16 bytes, the last of them with the tensors' end inside: behind it stand NaN,
    which must not reach any row."""
    g = gen(100 * rows + hidden)

    def ending_with_nan(n):
        flat = torch.full((n + 16,), float("nan"), dtype=dtype, device="cuda")
        flat[:n] = randn(g, n, dtype=dtype)
        return flat[:n]

    x, r = (ending_with_nan(rows * hidden).view(rows, hidden) for _ in range(2))
    w = 1 + randn(g, hidden, dtype=dtype, std=0.2)
    for residual in (None, r):
        check_norm(x, w, residual)


@pytest.mark.parametrize("rows,hidden,dtype", [(2500, 4096, BF16), (1500, 8191, F16), (900, 16383, F16)])
def test_norm_in_place_over_many_rows(rows, hidden, dtype):
    """h in the place of x or of the residual where a block has several rows, each read while the one
    before it is written."""
    g = gen(rows)
    x, r = randn(g, rows, hidden, dtype=dtype), randn(g, rows, hidden, dtype=dtype, std=4.0)
    w = 1 + randn(g, hidden, dtype=dtype, std=0.2)
    code = {F16: capi.DTYPE_F16, BF16: capi.DTYPE_BF16}[dtype]
    stream = torch.cuda.current_stream().cuda_stream
    y, h = ops.add_rms_norm(x, w, 1e-5, r)
    q, scales, _ = ops.add_rms_norm_quant(x, w, 1e-5, r)
    for place in range(2):
        for eight in (False, True):
            pair = [x.clone(), r.clone()]
            out, out_scales = torch.empty_like(q if eight else y), torch.empty_like(scales)
            args = (pair[place].data_ptr(), pair[0].data_ptr(), pair[1].data_ptr(), w.data_ptr(), 1e-5, code,
                    rows, hidden, stream)
            if eight:
                capi.call("int4gemv_add_rms_norm_quant", out.data_ptr(), out_scales.data_ptr(), *args)
                assert same_bits(out, q) and same_bits(out_scales, scales)
            else:
                capi.call("int4gemv_add_rms_norm", out.data_ptr(), *args)
                assert same_bits(out, y)
            assert same_bits(pair[place], h) and same_bits(pair[1 - place], (x, r)[1 - place])


# Tables for the kernel of small calls and, wider, for the one for any call.
WIDTHS = [24, 6000]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("group,dim", [(4, 64), (17, 128), (3, 256)])
def test_attention_of_refused_pages_gives_zeros(group, dim, weights, width):
    """Sequences whose pages are all outside of the cache, as in the padded slots of a captured batch:
    zeros, and nothing written; the others as they are without those."""
    c = Paged([1, 200, 0, 300, 40], 2, dim, 16, F16, seed=dim, width=width)
    q = randn(c.g, 5, 2 * group, dim, dtype=F16)
    k = randn(c.g, 5, 2, dim, dtype=F16)
    good = Paged([1, 200, 0, 300, 40], 2, dim, 16, F16, seed=dim, width=width)
    want = ops.paged_attention(q, good.k, good.v, good.table, good.seq_lens, 0.1, k, k,
                               good.weights if weights else None)
    table = c.table.clone()
    table[0], table[3], table[4, 1:] = -1, c.k.shape[0], 10**6
    before = c.k.clone(), c.v.clone(), c.weights.clone()
    out = ops.paged_attention(q, c.k, c.v, table, c.seq_lens, 0.1, k, k, c.weights if weights else None)
    assert capi.device_status() == capi.STATUS_BAD_PAGE
    assert (out[0] == 0).all() and (out[3] == 0).all() and (out[2] == 0).all()
    assert same_bits(out[1], want[1]) and out[4].isfinite().all()
    for b in (0, 3):  # the pages that these had are as they were
        pages, offs = ref.positions(c.table[b], c.lens[b], 16)
        assert same_bits(c.k[pages, offs], before[0][pages, offs])
        assert same_bits(c.v[pages, offs], before[1][pages, offs])
        assert same_bits(c.weights[pages, :, offs], before[2][pages, :, offs])
    empty = torch.empty(0, 16, 2, dim, dtype=F16, device="cuda")
    none = torch.empty(0, 2, 16, device="cuda")
    out = ops.paged_attention(q, empty, empty, c.table, c.seq_lens, 0.1, k, k, none if weights else None)
    assert capi.device_status() == capi.STATUS_BAD_PAGE
    assert (out == 0).all()


@pytest.mark.parametrize("width", WIDTHS)
def test_attention_of_scores_without_a_softmax(width):
    """Scores that are all -inf, a NaN or +inf among them: no softmax, so NaN, as the formula gives it;
    some of -inf count as 0."""
    c = Paged([20, 300, 300, 300, 300], 1, 64, 16, BF16, seed=1, width=width)
    q = torch.ones(5, 4, 64, dtype=BF16, device="cuda")
    at = [ref.positions(c.table[b], c.lens[b], 16) for b in range(5)]
    c.k[at[0]] = float("-inf")
    c.k[at[1]] = float("-inf")
    c.k[at[2][0][7], at[2][1][7]] = float("nan")
    c.k[at[3][0][299], at[3][1][299]] = float("inf")
    some = torch.arange(300) % 3 != 0
    c.k[at[4][0][some], at[4][1][some]] = float("-inf")
    out = ops.paged_attention(q, c.k, c.v, c.table, c.seq_lens, 0.125)
    assert out[:4].isnan().all()
    kept = ~some
    v = c.v[at[4][0][kept], at[4][1][kept], 0].double()
    s = c.k[at[4][0][kept], at[4][1][kept], 0].double().sum(-1) * 0.125
    p = torch.softmax(s, 0)
    # scores of up to 4: off by 64 / 16 + 2 additions at 2^-22 of 0.125 sum|k| <= 32, as in
    # ref.attention, and the pair of 16-bit numbers
    bound = (2 * (6 * 2.0**-22 * 32 + 2.0**-20) + 2.0**-16 + 530 * 2.0**-23) * (p @ v.abs()) + 2.0**-8 * (p @ v).abs()
    assert_within(out[4], (p @ v).expand(4, 64), bound.expand(4, 64))


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_far_below_a_peak(dtype, width):
    """One position takes nearly all of the probability and has a value of 0: the result is the sum of
    probabilities of 2^-25 each, which one 16-bit format or the other does not hold beside 1."""
    c = Paged([64, 100], 2, 64, 16, dtype, seed=3, width=width)
    q = torch.zeros(2, 6, 64, dtype=dtype, device="cuda")
    q[..., 0] = 1
    for b, n in enumerate(c.lens):
        pages, offs = ref.positions(c.table[b], n, 16)
        c.k[pages, offs], c.v[pages, offs] = 0, 1000
        c.k[pages[5], offs[5]], c.v[pages[5], offs[5]] = 17.4, 0
    out = ops.paged_attention(q, c.k, c.v, c.table, c.seq_lens, 1.0)
    want, bound, _, _ = ref.attention(q, c.k, c.v, c.table, c.lens, 1.0)
    # an fp16 probability is off by up to 2^-25, where the largest is at least 2^7
    tail = torch.tensor(c.lens, device="cuda")[:, None, None] * 2.0**-32 * 1000
    assert want.min() > 1e-3 and (tail < 0.02 * want).all()
    assert_within(out, want, bound + tail)


@pytest.mark.parametrize("batch,width", [(80, 24), (500, 6000)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_of_scores_whose_steps_are_wide(dtype, batch, width):
    """Scores of 2^27 (in base 2), whose neighbours are 16 apart: those of a later tile above the first
    one's by one step, and by less than the rise at which a warp takes a new reference plus a step."""
    c = Paged([300] * batch, 1, 64, 16, dtype, seed=4, width=width)
    c.k.zero_()
    pages, offs = ref.positions(c.table[0], 300, 16)
    for b in range(batch):
        pages, offs = ref.positions(c.table[b], 300, 16)
        c.k[pages, offs, 0, 0] = 2.0**15
        c.k[pages, offs, 0, 1] = 16.0
        c.k[pages[200:], offs[200:], 0, 1] = 32.0
    q = torch.zeros(batch, 2, 64, dtype=dtype, device="cuda")
    q[..., 0], q[..., 1] = 2.0**12, 1
    out = ops.paged_attention(q, c.k, c.v, c.table, c.seq_lens, 0.6931472)  # ln 2
    want, _, probs, _ = ref.attention(q, c.k, c.v, c.table, c.lens, 0.6931472)
    # the 100 later positions share all but 2^-15, whatever the rounding of the scores (a step off)
    # does to the rest
    for b in range(batch):
        pages, offs = ref.positions(c.table[b], 300, 16)
        v = c.v[pages[200:], offs[200:], 0].double()
        assert_within(out[b], v.mean(0).expand(2, 64), (ref.HALF[dtype] + 2.0**-12) * (v.abs().max() * 2).expand(2, 64))


@pytest.mark.parametrize("hkv,n", [(8, 1000), (3, 500), (8, 4000)])
def test_attention_of_clusters_around_what_runs_at_once(hkv, n):
    """One to five sequences: items on both sides of the number of clusters that run at once."""
    for batch in range(1, 6):
        check_attention(Paged([n - 7 * b for b in range(batch)], hkv, 128, 16, F16, seed=batch), 4 * hkv, F16,
                        True, True)


FIRST_CALL = """
import torch
from int4gemv import capi, ops
d = dict(device="cuda")
x, w = torch.randn(8, 512, **d).half(), torch.ones(512, **d).half()
q, kv = torch.randn(2, 4, 64, **d).half(), torch.randn(20, 16, 2, 64, **d).half()
v = kv.clone()
table = torch.arange(8, **d).int().view(2, 4)
new = torch.arange(8, 16, **d).int().view(2, 4)
lens = torch.tensor([60, 33], **d).int()
weights = torch.rand(20, 2, 16, **d)
tokens = torch.zeros(8, dtype=torch.int64, **d)

def calls():
    out = list(ops.add_rms_norm(x, w, 1e-5, x)) + list(ops.add_rms_norm_quant(x, w))
    out += [ops.paged_attention(q, kv, v, table, lens, 0.125), ops.paged_attention(q, kv, v, table, lens, 0.1)]
    out += ops.paged_evict(kv, v, weights, table, lens, new, 20, 5)
    out += list(ops.token_logprobs(x, tokens, 3)) + list(ops.token_logprobs(x, tokens, 0))
    return out

torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = calls()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, calls()))
assert capi.device_status() == 0
print("captured first")
"""


def test_the_first_call_of_a_process_may_be_captured():
    """Kernels are loaded and their limits set on first use, which a capture has to allow."""
    env = dict(os.environ, PYTHONPATH=str(Path(ops.LIBRARY_PATH).parents[1]))
    run = subprocess.run([sys.executable, "-c", FIRST_CALL], env=env, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "captured first" in run.stdout, run.stderr[-2000:]


@pytest.mark.parametrize("rows,hidden,dtype", [
    (1000, 4096, F16), (10000, 129, BF16), (6000, 64, F32), (20000, 7, F16),  # a chunk a thread, or one lane's
    (1000, 8192, BF16), (1000, 8191, F16), (900, 8192, F32), (2000, 2049, F32),  # two
    (700, 16383, F16), (600, 8301, F32),  # three
    (450, 16384, BF16), (400, 20000, F16)])  # two in whole rows, and the loop that reads a row twice
def test_norm_of_more_rows_than_blocks(rows, hidden, dtype):
    """Blocks of several rows: the next one is read while one is stored, rows that end inside 16 bytes,
    the tensors' end inside of the last ones."""
    g = gen(rows + hidden)
    x, w = randn(g, rows, hidden, dtype=dtype), 1 + randn(g, hidden, dtype=dtype, std=0.2)
    r = randn(g, rows, hidden, dtype=dtype, std=4.0)
    x[::7] *= 16  # rows of other sizes, whose statistics must not reach their neighbours
    for residual in (None, r):
        check_norm(x, w, residual)


def test_norm_writes_h_without_a_residual():
    """Through the C ABI h may be asked for without a residual: a copy of x, or x in its own place."""
    g = gen(2)
    x, w = randn(g, 300, 4096, dtype=BF16), randn(g, 4096, dtype=BF16)
    want, _ = ops.add_rms_norm(x, w, 1e-5)
    for h in (torch.empty_like(x), x):
        y, before = torch.empty_like(x), x.clone()
        capi.call("int4gemv_add_rms_norm", y.data_ptr(), h.data_ptr(), x.data_ptr(), None, w.data_ptr(), 1e-5,
                  capi.DTYPE_BF16, 300, 4096, torch.cuda.current_stream().cuda_stream)
        assert same_bits(h, before) and same_bits(x, before)
        # the loop that reads a row twice adds its squares in another order
        assert_within(y, want.double(), want.double().abs() * 2 * (ref.HALF[BF16] + ref.NORM_F32))


@pytest.mark.parametrize("rows,vocab,dtype", [(1300, 5003, F16), (1300, 5003, F32), (1500, 1001, BF16),
                                              (1200, 8192, F32), (700, 20000, F16)])
def test_logprobs_of_more_rows_than_blocks(rows, vocab, dtype):
    """Blocks of several rows, that begin at other places of 16 bytes, with and without alternatives."""
    g = gen(vocab)
    logits = randn(g, rows, vocab, dtype=dtype, std=3.0)
    logits[::5] += 20  # other maxima, and a mask, from row to row
    logits[::3, : vocab // 2] = float("-inf")
    tokens = torch.randint(vocab, (rows,), generator=g, device="cuda")
    for top in (0, 1, 7, 32):
        check_logprobs(logits, tokens, top)


@pytest.mark.parametrize("rows,hidden", [(400, 4096), (1000, 1001), (3, 30000)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_norm_of_values_whose_squares_pass_fp32(rows, hidden, dtype):
    """Rows whose sum of squares passes 2^128 give y = 0 and the least scale, those with an infinity NaN;
    h is right all the same, and so are the rows around them."""
    g = gen(rows * hidden)
    x, w = randn(g, rows, hidden, dtype=dtype), 1 + randn(g, hidden, dtype=dtype, std=0.2)
    r = randn(g, rows, hidden, dtype=dtype, std=4.0)
    x[::3, 5] = 1e20
    x[1::3, 6] = float("inf")
    y, h = ops.add_rms_norm(x, w, 1e-5, r)
    q, scales, h2 = ops.add_rms_norm_quant(x, w, 1e-5, r)
    assert same_bits(h, (x.double() + r.double()).to(dtype)) and same_bits(h, h2)
    assert (y[::3] == 0).all() and (q[::3].float() == 0).all() and (scales[::3] == 1e-12).all()
    assert scales[1::3].isnan().all() and y[1::3, 6].isnan().all()
    # a call of fewer rows may sum a row by more threads, in another order: compared with 64 bits
    want, _ = ref.norm(x[2::3], w, 1e-5, r[2::3])
    assert_within(y[2::3], want, want.abs() * (ref.HALF[dtype] + ref.NORM_F32))


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("group", [4, 17])
def test_attention_new_token_beyond_the_table(group, width):
    """The table's last position belongs to an earlier token, which the new one must not replace: the call
    is as without new tokens, and the status says so."""
    page = 16
    c = Paged([64, width * page, 100], 2, 64, page, F16, seed=9, width=width)
    q, k = randn(c.g, 3, 2 * group, 64, dtype=F16), randn(c.g, 3, 2, 64, dtype=F16)
    lens = c.seq_lens.clone()
    lens[1] += 3
    before = c.k.clone(), c.v.clone(), c.weights.clone()
    want = ops.paged_attention(q[1:2], c.k, c.v, c.table[1:2], c.seq_lens[1:2], 0.1, weights=c.weights)
    pages, offs = ref.positions(c.table[1], width * page, page)
    want_w = c.weights[pages, :, offs]
    for t, was in zip((c.k, c.v, c.weights), before):
        t.copy_(was)
    out = ops.paged_attention(q, c.k, c.v, c.table, lens, 0.1, k, k, c.weights)
    assert capi.device_status() == capi.STATUS_BAD_PAGE
    assert same_bits(c.k[pages, offs], before[0][pages, offs])
    assert same_bits(c.v[pages, offs], before[1][pages, offs])
    # another batch may split the sequence elsewhere: both are within the bound of the 64-bit result
    _, bound, probs, rel = ref.attention(q, c.k, c.v, c.table, c.lens, 0.1)
    assert_within(out[1:2], want.double(), 2 * bound[1:2])
    p = probs[1].sum(1).T
    bound_w = 2 * (p * (rel[1] + group * ref.F32) + (want_w.double() * 2 * ref.F32) + group * 2.0**-126)
    assert_within(c.weights[pages, :, offs], want_w.double(), bound_w)
    for b in (0, 2):  # the others got theirs
        pages, offs = ref.positions(c.table[b], c.lens[b], page)
        assert same_bits(c.k[pages[-1], offs[-1]], k[b])


@pytest.mark.parametrize("width", WIDTHS)
def test_captured_attention_follows_its_inputs(width):
    """One graph, replayed over lengths from nothing to the whole table, with pages, queries and new
    tokens of each: what a decode loop does."""
    c = Paged([300, 300, 300], 2, 128, 16, F16, seed=8, width=width)
    q, k = randn(c.g, 3, 8, 128, dtype=F16), randn(c.g, 3, 2, 128, dtype=F16)
    args = (q, c.k, c.v, c.table, c.seq_lens, 0.09, k, k, c.weights)
    ops.paged_attention(*args)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.paged_attention(*args)
    for lens in ((0, 0, 0), (1, 0, 300), (16, 17, 1), (128, 129, 255), (300, 64, 5)):
        c.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        q.copy_(randn(c.g, 3, 8, 128, dtype=F16))
        k.copy_(randn(c.g, 3, 2, 128, dtype=F16))
        c.table.copy_(c.table.roll(1, 0))
        before = c.k.clone(), c.v.clone(), c.weights.clone()
        g.replay()
        after = out.clone(), c.k.clone(), c.v.clone(), c.weights.clone()
        for t, was in zip((c.k, c.v, c.weights), before):
            t.copy_(was)
        want = ops.paged_attention(*args)
        assert all(same_bits(a, b) for a, b in zip(after, (want, c.k, c.v, c.weights)))
        assert all((out[b] == 0).all() for b in range(3) if lens[b] == 0)


@pytest.mark.parametrize("k_layout,v_layout", [("heads", "tokens"), ("tokens", "pairs")])
def test_caches_of_two_layouts(k_layout, v_layout):
    """Keys and values with strides of their own."""
    for width in WIDTHS:
        c = Paged([200, 77, 0, 31], 3, 64, 16, BF16, seed=2, layout=k_layout, width=width, spare=60)
        other = Paged([200, 77, 0, 31], 3, 64, 16, BF16, seed=2, layout=v_layout, width=width, spare=60)
        c.v = other.v
        assert c.k.stride() != c.v.stride()
        check_attention(c, 12, BF16, True, True)
        check_evict(c, 50, 9)


def test_pages_longer_than_sequences():
    """A contiguous cache: one page a sequence, of a size that is no power of two."""
    c = Paged([5000, 1, 3777], 2, 64, 5003, F16, seed=3, spare=3)
    check_attention(c, 10, F16, True, True)
    check_evict(c, 2500, 100)


def test_weights_that_are_not_aligned_to_four():
    """Weights whose first element is no multiple of 16 bytes, in pages of a multiple of four."""
    c = Paged([300, 90], 2, 64, 16, F16, seed=6, spare=40)
    flat = torch.empty(c.weights.numel() + 1, device="cuda")
    flat[1:] = c.weights.flatten()
    c.weights = flat[1:].view_as(c.weights)
    assert c.weights.data_ptr() % 16 == 4
    check_attention(c, 8, F16, True, True)
    check_evict(c, 100, 30)


# ---- Offsets behind 2^31 elements ----------------------------------------------------------------


def test_norm_of_far_rows():
    """Rows of a tensor of more than 2^31 elements, whole and odd."""
    for hidden, rows in ((8192, 2**18 + 300), (8191, 2**18 + 300)):
        x = torch.zeros(rows, hidden, dtype=BF16, device="cuda")
        g = gen(hidden)
        at = torch.tensor([0, 1, rows // 2, rows - 300, rows - 2, rows - 1], device="cuda")
        x[at] = randn(g, 6, hidden, dtype=BF16)
        w = 1 + randn(g, hidden, dtype=BF16, std=0.2)
        assert x.numel() > 2**31
        want, _ = ref.norm(x[at], w, 1e-5)
        y, _ = ops.add_rms_norm(x, w)
        assert_within(y[at], want, want.abs() * (ref.HALF[BF16] + ref.NORM_F32))
        assert not y[rows - 3].any()


def test_evict_of_far_pages():
    """Old and new pages whose elements lie behind 2^31 elements."""
    per_page = 16 * 2 * 128
    c = Paged([300, 90], 2, 128, 16, F16, seed=6, spare=40, first_page=2**31 // per_page + 5)
    assert c.k.stride(0) * c.table.max().item() > 2**31
    check_evict(c, 100, 30)


def test_logprobs_of_far_rows():
    """Rows that lie 2^30 elements apart."""
    flat = torch.empty(3 * 2**30 + 6000, dtype=F16, device="cuda")
    logits = flat.as_strided((4, 5000), (2**30 + 1, 1))
    g = gen(7)
    for i in range(4):
        logits[i] = randn(g, 5000, dtype=F16, std=3.0)
    check_logprobs(logits, torch.tensor([0, 4999, 17, 2500], device="cuda"), 6)
