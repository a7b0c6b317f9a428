"""The decode-step operators on a B200 against their plain 64-bit forms (decode_reference.py)."""

import ctypes
import math

import pytest
import torch

import decode_reference as ref
from int4gemv import capi, ops

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def no_status_left():
    yield
    assert capi.device_status() == 0


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def same_bits(a, b):
    return a.dtype == b.dtype and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def assert_within(got, want, bound, what=""):
    assert got.shape == want.shape
    if not got.numel():
        return
    off = (got.double() - want).abs()
    worst = (off / bound.clamp_min(1e-300)).max().item()
    inside = bool((off <= bound).all())
    assert inside, f"{what}: error up to {worst:.3g} of its bound"


# ---- add_rms_norm --------------------------------------------------------------------------------

NORM_SHAPES = [(1, 1), (1, 4096), (5, 7), (130, 64), (6, 129), (3, 1000), (37, 8192), (2, 8191),
               (3, 16384), (2, 40000), (2, 33333)]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,hidden", NORM_SHAPES)
def test_norm(rows, hidden, dtype):
    g = gen(hidden)
    x, w = randn(g, rows, hidden, dtype=dtype), 1 + randn(g, hidden, dtype=dtype, std=0.2)
    r = randn(g, rows, hidden, dtype=dtype, std=4.0)
    for residual in (None, r):
        want, h64 = ref.norm(x, w, 1e-5, residual)
        y, h = ops.add_rms_norm(x, w, 1e-5, residual)
        tiny = 2.0**-25 if dtype == F16 else 0.0
        assert_within(y, want, want.abs() * (ref.HALF[dtype] + ref.NORM_F32) + tiny, "y")
        assert_within(h, h64, h64.abs() * (ref.HALF[dtype] + ref.F32) + tiny, "h")
        q, scales, h2 = ops.add_rms_norm_quant(x, w, 1e-5, residual)
        assert q.dtype == torch.float8_e4m3fn and scales.dtype == F32 and same_bits(h, h2)
        s64 = want.abs().amax(-1) / 448
        assert_within(scales, s64, s64 * (ref.NORM_F32 + 4 * ref.F32), "scales")
        v = want / s64[:, None]
        # half a step of e4m3: 2^-4 of the value, 2^-10 below 2^-6
        assert_within(q.float(), v, v.abs() * (2.0**-4 + 2 * ref.NORM_F32) + 2.0**-10, "q")


def test_norm_special_rows():
    """Rows of zeros, and rows with a NaN or infinity, do not disturb others."""
    x = torch.ones(4, 512, dtype=F16, device="cuda")
    x[0] = 0
    x[1, 7] = float("nan")
    x[2, 9] = float("inf")
    w = torch.ones(512, dtype=F16, device="cuda")
    y, _ = ops.add_rms_norm(x, w, 1e-5)
    assert (y[0] == 0).all() and y[1].isnan().all() and y[2, 9].isnan() and (y[2, :9] == 0).all()
    assert torch.equal(y[3], ops.add_rms_norm(x[3:], w, 1e-5)[0][0])
    q, scales, _ = ops.add_rms_norm_quant(x, w, 1e-5)
    assert scales[0].item() == pytest.approx(1e-12) and (q[0].float() == 0).all()
    assert scales[1:3].isnan().all() and q[1].float().isnan().all() and not q[3].float().isnan().any()


@pytest.mark.parametrize("hidden,shift", [(1024, 1), (1024, 4), (77, 3)])
def test_norm_unaligned_tensors(hidden, shift):
    """Tensors that start inside a 16-byte chunk, each at another place."""
    g = gen(3)
    def at(rows, off):
        flat = randn(g, rows * hidden + 16, dtype=F16)
        return flat[off:off + rows * hidden].view(rows, hidden)
    x, r, w = at(5, shift), at(5, 0), at(1, 2)[0]
    want, _ = ref.norm(x, w, 1e-5, r)
    y, h = ops.add_rms_norm(x, w, 1e-5, r)
    assert_within(y, want, want.abs() * (ref.HALF[F16] + ref.NORM_F32) + 2.0**-25)
    assert same_bits(h, (x.float() + r.float()).half())


def test_norm_in_place_through_c_abi():
    """h may be the residual or x itself."""
    g = gen(5)
    for hidden in (4096, 33000, 100):
        x, r, w = randn(g, 6, hidden, dtype=BF16), randn(g, 6, hidden, dtype=BF16), randn(g, hidden, dtype=BF16)
        y, h = ops.add_rms_norm(x, w, 1e-6, r)
        for target in (x.clone(), r.clone()):
            a = target if torch.equal(target, x) else x
            b = target if torch.equal(target, r) else r
            out = torch.empty_like(x)
            capi.call("int4gemv_add_rms_norm", out.data_ptr(), target.data_ptr(), a.data_ptr(),
                      b.data_ptr(), w.data_ptr(), 1e-6, capi.DTYPE_BF16, 6, hidden,
                      torch.cuda.current_stream().cuda_stream)
            assert same_bits(out, y) and same_bits(target, h)


def test_norm_refusals():
    x = torch.zeros(4, 64, dtype=F16, device="cuda")
    for call, message in (
            (lambda: ops.add_rms_norm(x.t(), x[0]), "contiguous 2-D CUDA"),
            (lambda: ops.add_rms_norm(x.to(torch.int32), x[0]), "float32, float16 or bfloat16"),
            (lambda: ops.add_rms_norm(x, x[0, :32].clone()), "weight must be a contiguous Half"),
            (lambda: ops.add_rms_norm(x, x[0].float()), "weight must be a contiguous Half"),
            (lambda: ops.add_rms_norm(x, x[0], 1e-5, x[:2]), "residual must be a contiguous Half"),
            (lambda: ops.add_rms_norm(x, x[0].cpu()), "weight must be")):
        with pytest.raises(RuntimeError, match=message):
            call()
    y, h = ops.add_rms_norm(x[:0], x[0])
    assert y.shape == (0, 64) and h.shape == (0, 64)


# ---- paged_attention -----------------------------------------------------------------------------


class Paged:
    """A cache whose unused places hold NaN and infinities, with tables of scattered pages."""

    def __init__(self, lens, hkv, dim, page, dtype, seed, layout="tokens", width=None, spare=3,
                 first_page=0):
        g = gen(seed)
        self.lens, self.page, self.hkv, self.dim = lens, page, hkv, dim
        need = [-(-n // page) for n in lens]
        self.width = width or max(need + [1])
        total = sum(need) + spare
        blocks = first_page + total
        if layout == "tokens":
            kv = torch.empty(2, blocks, page, hkv, dim, dtype=dtype, device="cuda")
            self.k, self.v = kv[0], kv[1]
        elif layout == "heads":
            kv = torch.empty(2, blocks, hkv, page, dim, dtype=dtype, device="cuda")
            self.k, self.v = kv[0].transpose(1, 2), kv[1].transpose(1, 2)
        else:  # one tensor, the halves of each page
            kv = torch.empty(blocks, 2, page, hkv, dim, dtype=dtype, device="cuda")
            self.k, self.v = kv[:, 0], kv[:, 1]
        order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)) + first_page
        self.table = torch.full((len(lens), self.width), -7, dtype=torch.int32)
        self.k[first_page:] = float("nan")
        self.v[first_page:] = float("inf")
        at = 0
        for b, n in enumerate(lens):
            self.table[b, :need[b]] = order[at:at + need[b]].int()
            at += need[b]
            if n:
                pages, offs = ref.positions(self.table[b], n, page)
                self.k[pages, offs] = randn(g, n, hkv, dim, dtype=dtype)
                self.v[pages, offs] = randn(g, n, hkv, dim, dtype=dtype)
        self.spare_pages = order[at:]
        self.weights = torch.rand(blocks, hkv, page, generator=g, device="cuda")
        self.table = self.table.cuda()
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.g = g


def check_attention(c, hq, dtype, append, weights, scale=None):
    batch = len(c.lens)
    scale = 1 / math.sqrt(c.dim) if scale is None else scale
    q = randn(c.g, batch, hq, c.dim, dtype=dtype, std=1.5)
    k = randn(c.g, batch, c.hkv, c.dim, dtype=dtype) if append else None
    v = randn(c.g, batch, c.hkv, c.dim, dtype=dtype) if append else None
    after_k, after_v = c.k.clone(), c.v.clone()
    after_w = c.weights.double()
    w = c.weights if weights else None
    if append:
        for b, n in enumerate(c.lens):
            if n:
                pages, offs = ref.positions(c.table[b], n, c.page)
                after_k[pages[-1], offs[-1]] = k[b]
                after_v[pages[-1], offs[-1]] = v[b]
                # what the page held there before must not reach anything
                c.k[pages[-1], offs[-1]] = float("nan")
                c.v[pages[-1], offs[-1]] = float("nan")
                if weights:
                    c.weights[pages[-1], :, offs[-1]] = float("nan")
                    after_w[pages[-1], :, offs[-1]] = 0
    out = ops.paged_attention(q, c.k, c.v, c.table, c.seq_lens, scale, k, v, w)
    want, bound, probs, rel = ref.attention(q, after_k, after_v, c.table, c.lens, scale)
    assert_within(out, want, bound, "out")
    assert same_bits(c.k, after_k) and same_bits(c.v, after_v)
    if not weights:
        return
    group = hq // c.hkv
    bound_w = torch.zeros_like(after_w)
    for b, n in enumerate(c.lens):
        if n:
            pages, offs = ref.positions(c.table[b], n, c.page)
            p = probs[b].sum(1).T  # [n, hkv]
            after_w[pages, :, offs] += p
            bound_w[pages, :, offs] = p * (rel[b] + group * ref.F32)
    # each probability below fp32's smallest normal number, 2^-126, is 0 in the kernel: up to that
    # much off, once for each query head of the group
    bound_w += after_w * 2 * ref.F32 + group * 2.0**-126
    assert_within(c.weights, after_w, bound_w, "weights")


LENS = [1, 0, 15, 16, 17, 63, 64, 65, 200, 333]


SHAPES = [
    (4, 2, 128, 16, "tokens"), (4, 2, 128, 16, "heads"), (8, 2, 128, 32, "pairs"),
    (1, 3, 64, 16, "tokens"), (2, 1, 64, 8, "heads"), (3, 2, 80, 48, "pairs"),
    (7, 1, 96, 64, "tokens"), (16, 2, 128, 128, "heads"), (17, 1, 64, 16, "tokens"),
    (40, 1, 128, 16, "pairs"), (5, 2, 256, 16, "tokens"), (16, 1, 192, 24, "heads"),
    (4, 2, 8, 1, "tokens"), (6, 2, 40, 5, "heads"), (33, 1, 136, 256, "tokens"),
]


@pytest.mark.parametrize("group,hkv,dim,page,layout", SHAPES)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention(group, hkv, dim, page, layout, dtype):
    for append, weights in ((False, False), (True, True)):
        c = Paged(LENS, hkv, dim, page, dtype, seed=group * dim, layout=layout, width=400)
        check_attention(c, group * hkv, dtype, append, weights)


@pytest.mark.parametrize("group,hkv,dim,page,layout", SHAPES)
def test_attention_of_narrow_and_wide_tables(group, hkv, dim, page, layout):
    """The same call by the kernel for small calls (a narrow table, few sequences) and by the one for
    any call (a table too wide for it), each with new tokens and weights."""
    for width in (-(-333 // page), 60000 // page):
        c = Paged([333, 0, 64, 65], hkv, dim, page, F16, seed=dim + page, layout=layout, width=width)
        check_attention(c, group * hkv, F16, True, True)


@pytest.mark.parametrize("lens,group,hkv,dim", [
    ([70001], 4, 1, 128), ([40000, 1, 0, 900], 8, 2, 64), ([1], 4, 8, 128), ([20011], 1, 1, 256),
    ([5] * 300 + [0] * 200 + [700] * 20, 2, 2, 64), ([0, 0], 4, 2, 128),
    ([64 * i for i in range(20)], 20, 1, 64)])
def test_attention_lengths(lens, group, hkv, dim):
    """Long sequences that many blocks share, more sequences than a block has threads, none at all."""
    for append, weights in ((True, False), (False, True)):
        check_attention(Paged(lens, hkv, dim, 16, F16, seed=len(lens)), group * hkv, F16, append, weights)


def test_attention_peaked_scores():
    """Scores of hundreds (one position takes all), of both signs."""
    for scale in (30.0, -30.0, 0.0):
        check_attention(Paged([300, 90], 2, 64, 16, BF16, seed=5), 8, BF16, True, True, scale=scale)


def test_attention_far_offsets():
    """Pages whose elements lie behind 2^32 bytes and 2^31 elements."""
    per_page = 16 * 2 * 128
    c = Paged([100, 33], 2, 128, 16, F16, seed=9, first_page=2**31 // per_page + 5)
    assert c.k.stride(0) * c.table.max().item() > 2**31
    check_attention(c, 8, F16, True, True)


def test_attention_is_deterministic_and_takes_views():
    """The same bits every time, whatever ran before in the workspace, and from a q that is a row
    range of a larger tensor."""
    c = Paged([5000, 17, 1200], 2, 128, 16, F16, seed=2)
    q = randn(c.g, 6, 8, 128, dtype=F16)[2:5]
    first = ops.paged_attention(q, c.k, c.v, c.table, c.seq_lens, 0.1)
    for _ in range(3):
        junk = torch.full((1 << 22,), float("nan"), device="cuda")
        del junk
        assert same_bits(first, ops.paged_attention(q, c.k, c.v, c.table, c.seq_lens, 0.1))


@pytest.mark.parametrize("width", [7, 5000])
def test_bad_pages_and_lengths_are_reported(width):
    """A page outside of the cache is left out, a length the table has no room for clamped: the
    status says so, other sequences and everything outside of the call's places stay as they were."""
    c = Paged([100, 80, 64], 2, 64, 16, F16, seed=4, width=width)
    q = randn(c.g, 3, 4, 64, dtype=F16)
    good = ops.paged_attention(q, c.k, c.v, c.table, c.seq_lens, 0.125)
    k0, v0, w0 = c.k.clone(), c.v.clone(), c.weights.clone()
    table = c.table.clone()
    table[0, 2], table[0, 4] = 10**9, -1
    out = ops.paged_attention(q, c.k, c.v, table, c.seq_lens, 0.125, weights=c.weights)
    assert capi.device_status() == capi.STATUS_BAD_PAGE
    assert same_bits(out[1:], good[1:])
    keep = [j for j in range(100) if j // 16 not in (2, 4)]
    pages, offs = ref.positions(c.table[0], 100, 16)
    pages, offs = pages[keep], offs[keep]
    s = torch.einsum("hgd,nhd->hgn", q[0].double().view(2, 2, 64), c.k[pages, offs].double()) * 0.125
    want = torch.einsum("hgn,nhd->hgd", torch.softmax(s, -1), c.v[pages, offs].double()).reshape(4, 64)
    # |s| below 20 here: the bound of attention() with room
    assert_within(out[0], want, want.abs() * 2.0**-11 + 2.0**-13)
    assert same_bits(c.k, k0) and same_bits(c.v, v0)
    untouched = torch.ones_like(w0, dtype=torch.bool)
    for b in range(3):
        pages, offs = ref.positions(c.table[b], c.lens[b], 16)
        untouched[pages, :, offs] = False
    assert torch.equal(c.weights[untouched], w0[untouched])

    lens = torch.tensor([10**6, -3, 64], dtype=torch.int32, device="cuda")
    full = c.table.clone()
    full[0] = c.table[0, 0]  # the same page again and again
    out = ops.paged_attention(q, c.k, c.v, full, lens, 0.125)
    assert capi.device_status() == capi.STATUS_BAD_PAGE
    assert (out[1] == 0).all() and same_bits(out[2], good[2]) and out[0].isfinite().all()
    # the new token of a bad page is written nowhere
    new = randn(c.g, 3, 2, 64, dtype=F16)
    table = c.table.clone()
    table[1, 4] = c.k.shape[0]
    ops.paged_attention(q[1:2], c.k, c.v, table[1:2], c.seq_lens[1:2], 0.125, new[:1], new[:1])
    assert capi.device_status() == capi.STATUS_BAD_PAGE
    assert same_bits(c.k, k0) and same_bits(c.v, v0)
    empty = torch.empty(0, 16, 2, 64, dtype=F16, device="cuda")
    ops.paged_attention(q, empty, empty, c.table, c.seq_lens, 0.125)
    assert capi.device_status() == capi.STATUS_BAD_PAGE


def test_attention_no_pages_and_empty_batch():
    c = Paged([40], 2, 64, 16, F16, seed=4)
    q = randn(c.g, 1, 4, 64, dtype=F16)
    none = torch.empty(1, 0, dtype=torch.int32, device="cuda")
    out = ops.paged_attention(q, c.k, c.v, none, torch.zeros_like(c.seq_lens), 0.125)
    assert (out == 0).all()
    out = ops.paged_attention(q[:0], c.k, c.v, c.table[:0], c.seq_lens[:0], 0.125)
    assert out.shape == (0, 4, 64)


def test_attention_refusals():
    c = Paged([40, 3], 2, 64, 16, F16, seed=4)
    q = randn(c.g, 2, 4, 64, dtype=F16)
    k = randn(c.g, 2, 2, 64, dtype=F16)

    def call(q=q, kc=c.k, vc=c.v, table=c.table, lens=c.seq_lens, **more):
        return ops.paged_attention(q, kc, vc, table, lens, 0.125, **more)

    for run, message in (
            (lambda: call(q=q.bfloat16()), "q must be a contiguous Half"),
            (lambda: call(q=q[:, :3].contiguous()), "multiple of kv_heads"),
            (lambda: call(q=q.transpose(1, 2).contiguous()), "q must be"),
            (lambda: call(kc=c.k.float(), vc=c.v.float()), "float16 or bfloat16"),
            (lambda: call(vc=c.v.bfloat16()), "v_cache must be like k_cache"),
            (lambda: call(kc=c.k.transpose(2, 3), vc=c.v.transpose(2, 3)), "must be contiguous"),
            (lambda: call(table=c.table.long()), "block_table must be a contiguous Int"),
            (lambda: call(table=c.table[:1]), "block_table must be"),
            (lambda: call(lens=c.seq_lens.long()), "seq_lens must be a contiguous Int"),
            (lambda: call(lens=c.seq_lens.cpu()), "seq_lens must be"),
            (lambda: call(k=k), "k and v come together"),
            (lambda: call(k=k[:1], v=k[:1]), "k must be a contiguous Half"),
            (lambda: call(weights=c.weights.half()), "weights must be a contiguous Float"),
            (lambda: call(weights=c.weights[:-1]), "weights must be"),
            (lambda: call(kc=c.k[..., :60], vc=c.v[..., :60], q=q[..., :60].contiguous()), "head_dim 60"),
            (lambda: call(kc=c.k[..., 4:44], vc=c.v[..., 4:44], q=q[..., :40].contiguous()),
             "16-byte aligned")):
        with pytest.raises(RuntimeError, match=message):
            run()


def test_attention_through_c_abi():
    """Raw pointers and a caller's workspace; strides of head-major pages."""
    c = Paged([300, 20], 2, 64, 16, BF16, seed=8, layout="heads")
    q = randn(c.g, 2, 6, 64, dtype=BF16)
    want = ops.paged_attention(q, c.k, c.v, c.table, c.seq_lens, 0.125)
    pc = capi.PagedCache(k=c.k.data_ptr(), v=c.v.data_ptr(), num_blocks=c.k.shape[0], block_size=16,
                         kv_heads=2, head_dim=64, dtype=capi.DTYPE_BF16)
    for i in range(3):
        pc.k_strides[i], pc.v_strides[i] = c.k.stride(i), c.v.stride(i)
    size = capi.lib().int4gemv_paged_attention_workspace_size(ctypes.addressof(pc), 2, 6, c.width, 0)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    capi.call("int4gemv_paged_attention", out.data_ptr(), q.data_ptr(), ctypes.addressof(pc),
              c.table.data_ptr(), c.seq_lens.data_ptr(), 0.125, None, None, 0, 2, 6, c.width,
              ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
    assert same_bits(out, want)


# ---- paged_evict ---------------------------------------------------------------------------------


def check_evict(c, budget, recent, new_table=None):
    batch = len(c.lens)
    need = [-(-min(n, budget) // c.page) for n in c.lens]
    if new_table is None:
        new_table = torch.full((batch, -(-budget // c.page) + 1), -3, dtype=torch.int32)
        pages = c.spare_pages[:sum(need)].tolist()
        assert len(pages) == sum(need)
        for b in range(batch):
            new_table[b, :need[b]] = torch.tensor([pages.pop() for _ in range(need[b])], dtype=torch.int32)
        new_table = new_table.cuda()
    want_kept, want_lens = ref.evict(c.weights, c.table, c.lens, c.page, budget, recent)
    k, v, w = c.k.clone(), c.v.clone(), c.weights.clone()
    heads = torch.arange(c.hkv)
    for b, n in enumerate(c.lens):
        m = min(n, budget)
        if not m:
            continue
        src = want_kept[b, :, :m].long()
        pages, offs = c.table[b].cpu().long()[src // c.page], src % c.page  # [hkv, m]
        to_p, to_o = ref.positions(new_table[b], m, c.page)
        k[to_p[None], to_o[None], heads[:, None]] = c.k[pages, offs, heads[:, None]]
        v[to_p[None], to_o[None], heads[:, None]] = c.v[pages, offs, heads[:, None]]
        w[to_p[None], heads[:, None], to_o[None]] = c.weights[pages, heads[:, None], offs]
    kept, lens = ops.paged_evict(c.k, c.v, c.weights, c.table, c.seq_lens, new_table, budget, recent)
    assert kept.dtype == torch.int32 and torch.equal(kept.cpu(), want_kept)
    assert lens.dtype == torch.int32 and torch.equal(lens.cpu(), want_lens)
    # everything else is left as it was
    assert same_bits(c.k, k) and same_bits(c.v, v) and same_bits(c.weights, w)


@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (50, 0), (50, 50), (64, 10), (100, 31),
                                           (299, 5), (300, 5), (1000, 100)])
@pytest.mark.parametrize("layout", ["tokens", "heads", "pairs"])
def test_evict(budget, recent, layout):
    c = Paged([0, 1, 50, 51, 64, 300, 100], 3, 64, 16, F16, seed=budget, layout=layout, spare=200)
    check_evict(c, budget, recent)


@pytest.mark.parametrize("dim,page,hkv,dtype", [(8, 1, 1, F16), (80, 48, 2, BF16), (256, 8, 2, F16),
                                                (136, 7, 5, BF16), (64, 16, 4, F16), (128, 32, 8, BF16),
                                                (72, 16, 12, F16)])
def test_evict_shapes(dim, page, hkv, dtype):
    check_evict(Paged([200, 77, 30], hkv, dim, page, dtype, seed=dim, spare=400), 60, 20)


def test_evict_ties_and_special_weights():
    """Equal weights (the first positions stay), zeros of both signs, NaN, infinities, negatives."""
    for kind in range(5):
        c = Paged([400, 130], 2, 8, 16, F16, seed=kind, spare=60)
        w = c.weights
        if kind == 0:
            w.fill_(1.5)
        elif kind == 1:
            w.copy_((w * 3).floor())
        elif kind == 2:
            w.copy_(torch.where(w < 0.5, 0.0, -0.0))
        elif kind == 3:
            w[w < 0.1] = float("nan")
            w[w > 0.9] = float("inf")
            w[(w > 0.4) & (w < 0.5)] = float("-inf")
        else:
            w.sub_(0.5).mul_(1e-38)
        check_evict(c, 100, 30)


@pytest.mark.parametrize("n", [5000, 49153, 70000])
def test_evict_long(n):
    """More positions than a block keeps in shared memory."""
    c = Paged([n, 3000], 1, 8, 64, F16, seed=n, spare=400)
    check_evict(c, 10001, 501)


def test_evict_shared_prefix():
    """Two sequences whose first pages are the same: the old pages stay as they were."""
    c = Paged([200, 200], 2, 64, 16, F16, seed=1, spare=40)
    c.table[1, :6] = c.table[0, :6]
    check_evict(c, 70, 20)


def test_evict_bad_pages():
    c = Paged([100, 90], 2, 64, 16, F16, seed=3, spare=20)
    spare = c.spare_pages.int().cuda()
    new = torch.stack([spare[:4], spare[4:8]])
    good_kept, _ = ops.paged_evict(c.k, c.v, c.weights, c.table, c.seq_lens, new, 60, 20)
    k1, w1 = c.k.clone(), c.weights.clone()
    table, bad_new = c.table.clone(), new.clone()
    table[0, 1], bad_new[1, 2] = 10**6, -5
    kept, lens = ops.paged_evict(c.k, c.v, c.weights, table, c.seq_lens, bad_new, 60, 20)
    assert capi.device_status() == capi.STATUS_BAD_PAGE
    assert torch.equal(kept[1], good_kept[1]) and lens.tolist() == [60, 60]
    other = torch.ones(c.k.shape[0], dtype=torch.bool)
    other[new[0].cpu().long()] = False
    assert same_bits(c.k[other], k1[other]) and same_bits(c.weights[other], w1[other])


def test_evict_refusals_and_empty():
    c = Paged([100, 90], 2, 64, 16, F16, seed=3, spare=20)
    new = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    for run, message in (
            (lambda: ops.paged_evict(c.k, c.v, c.weights, c.table, c.seq_lens, new, 65, 0), "room for 64"),
            (lambda: ops.paged_evict(c.k, c.v, c.weights, c.table, c.seq_lens, new, 10, 11), "recent 11"),
            (lambda: ops.paged_evict(c.k, c.v, c.weights, c.table, c.seq_lens, new, 0, 0), "budget 0"),
            (lambda: ops.paged_evict(c.k, c.v, c.weights, c.table, c.seq_lens, new[:1], 10, 1), "new_table"),
            (lambda: ops.paged_evict(c.k, c.v, c.weights.double(), c.table, c.seq_lens, new, 10, 1),
             "weights must be")):
        with pytest.raises(RuntimeError, match=message):
            run()
    kept, lens = ops.paged_evict(c.k, c.v, c.weights, c.table[:0], c.seq_lens[:0], new[:0], 10, 1)
    assert kept.shape == (0, 2, 10) and lens.shape == (0,)
    none = torch.empty(2, 0, dtype=torch.int32, device="cuda")
    kept, lens = ops.paged_evict(c.k, c.v, c.weights, none, c.seq_lens * 0, new, 10, 1)
    assert (kept == -1).all() and lens.tolist() == [0, 0]


# ---- token_logprobs ------------------------------------------------------------------------------


def check_logprobs(logits, tokens, top):
    (lp, ent, top_lp, ids), off, off_ent = ref.logprobs(logits, tokens, top)
    got = ops.token_logprobs(logits, tokens, top)
    assert [t.dtype for t in got] == [F32, F32, F32, torch.int64]
    assert torch.equal(got[3], ids), (got[3] - ids).abs().max()
    for a, b, bound, what in ((got[0], lp, off, "logprobs"), (got[1], ent, off_ent, "entropy"),
                              (got[2], top_lp, off[:, None], "top")):
        fine = torch.isfinite(b)
        assert torch.equal(a[~fine].isnan(), b[~fine].isnan()) and torch.equal(torch.isfinite(a), fine), what
        bound = bound.expand(b.shape)
        assert_within(a[fine], b[fine], bound[fine], what)


@pytest.mark.parametrize("rows,vocab,dtype,top", [
    (1, 32001, F16, 5), (1, 128256, BF16, 32), (64, 32000, F16, 20), (3, 1, F16, 1), (2, 2, BF16, 2),
    (5, 31, F32, 31), (7, 1000, F32, 0), (300, 5003, BF16, 7), (2, 262144, F32, 32), (33, 4097, F16, 32),
    (150, 50257, F32, 3), (1, 700001, F16, 8)])
def test_logprobs(rows, vocab, dtype, top):
    g = gen(vocab)
    logits = randn(g, rows, vocab, dtype=dtype, std=3.0)
    tokens = torch.randint(vocab, (rows,), generator=g, device="cuda")
    check_logprobs(logits, tokens, top)
    # a peak that takes nearly all, and a grammar's mask
    logits[:, vocab // 2] = 40.0
    logits[torch.rand(rows, vocab, generator=g, device="cuda") < 0.7] = float("-inf")
    logits[:, vocab // 3] = 2.0
    check_logprobs(logits, tokens, top)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_logprobs_special_rows(dtype):
    """Each row beside ordinary ones: equal logits, rising, falling, the type's lowest value, -inf,
    NaN, +inf, all but a few masked, the only unmasked ones at the end, huge values."""
    vocab, top = 20000, 17
    g = gen(1)
    x = randn(g, 14, vocab, dtype=dtype)
    lowest = torch.finfo(dtype).min
    x[0] = 1.25
    x[1] = torch.linspace(-20, 20, vocab, device="cuda").to(dtype)
    x[2] = torch.linspace(20, -20, vocab, device="cuda").to(dtype)
    x[3] = lowest
    x[4, 5:] = lowest
    x[5] = float("-inf")
    x[6, 100] = float("nan")
    x[7, 200] = float("inf")
    x[8] = float("-inf")
    x[8, [3, 19999, 500]] = torch.tensor([1.0, 2.0, 2.0], device="cuda", dtype=dtype)
    x[9, :19000] = float("-inf")
    x[10] = 60000.0
    x[11] = 0
    x[11, ::2] = -0.0
    x[12, 7] = float("nan")
    x[12, 10:] = float("nan")
    tokens = torch.tensor([0, 19999, 0, 5, 2, 9, 7, 200, 500, 3, 1, 2, 7, 10], device="cuda")
    check_logprobs(x, tokens, top)
    check_logprobs(x, tokens, 0)
    check_logprobs(x, tokens, 32)
    # many rows, of which a block takes one after the other
    check_logprobs(x.repeat(60, 1), tokens.repeat(60), 17)


def test_logprobs_tokens_outside_and_views():
    g = gen(6)
    wide = randn(g, 6, 4100, dtype=F16, std=2.0)
    for logits in (wide[:, :4000], wide[1:4, 3:1000], wide[::2, 1:], wide[2:3]):
        rows, vocab = logits.shape
        tokens = torch.tensor([-1, vocab, 5, vocab - 1, 0, -100][:rows], device="cuda")
        check_logprobs(logits, tokens, 4)
    out = ops.token_logprobs(wide[:0], torch.zeros(0, dtype=torch.int64, device="cuda"), 3)
    assert [t.shape for t in out] == [(0,), (0,), (0, 3), (0, 3)]


def test_logprobs_refusals():
    x = torch.zeros(2, 100, dtype=F16, device="cuda")
    t = torch.zeros(2, dtype=torch.int64, device="cuda")
    for run, message in ((lambda: ops.token_logprobs(x, t.int()), "tokens must be a contiguous Long"),
                         (lambda: ops.token_logprobs(x, t[:1]), "tokens must be"),
                         (lambda: ops.token_logprobs(x.t(), t), "contiguous"),
                         (lambda: ops.token_logprobs(x.double(), t), "float32, float16 or bfloat16"),
                         (lambda: ops.token_logprobs(x, t, 33), "top 33"),
                         (lambda: ops.token_logprobs(x[:, :3], t, 4), "top 4"),
                         (lambda: ops.token_logprobs(x, t, -1), "top -1")):
        with pytest.raises(RuntimeError, match=message):
            run()


# ---- all of them: streams, graphs ----------------------------------------------------------------


def every_operator(seed):
    """A callable that runs all operators on its own inputs and returns their outputs."""
    c = Paged([3000, 17, 0, 500], 2, 64, 16, F16, seed=seed, spare=80)
    q, k = randn(c.g, 4, 8, 64, dtype=F16), randn(c.g, 4, 2, 64, dtype=F16)
    x, w = randn(c.g, 40, 4096, dtype=F16), randn(c.g, 4096, dtype=F16)
    logits = randn(c.g, 5, 30001, dtype=F16)
    tokens = torch.arange(5, device="cuda")
    new = c.spare_pages[:28].int().view(4, 7).cuda()
    first = c.k.clone(), c.v.clone(), c.weights.clone()

    def run():
        for t, was in zip((c.k, c.v, c.weights), first):
            t.copy_(was)
        out = [ops.paged_attention(q, c.k, c.v, c.table, c.seq_lens, 0.125, k, k, c.weights)]
        out += ops.paged_evict(c.k, c.v, c.weights, c.table, c.seq_lens, new, 100, 20)
        out += ops.add_rms_norm(x, w, 1e-5, x)
        out += ops.add_rms_norm_quant(x, w, 1e-5)
        out += ops.token_logprobs(logits, tokens, 9)
        return out + [c.k, c.v, c.weights]

    return run


def test_two_streams_at_once():
    runs = [every_operator(s) for s in (1, 2)]
    want = [[t.clone() for t in run()] for run in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in runs]
    got = [None, None]
    for _ in range(5):
        for i, run in enumerate(runs):
            with torch.cuda.stream(streams[i]):
                got[i] = run()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(same_bits(x, y) for x, y in zip(a, b))


def test_captured_graphs_replayed_at_once():
    runs = [every_operator(s) for s in (3, 4)]
    want = [[t.clone() for t in run()] for run in runs]
    graphs, outs = [], []
    for run in runs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in runs]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, want):
        assert all(same_bits(x, y) for x, y in zip(a, b))


@pytest.mark.skipif("torch.cuda.device_count() < 2")
def test_other_device():
    x, w = torch.randn(3, 512, device="cuda:1").half(), torch.ones(512, device="cuda:1").half()
    y, _ = ops.add_rms_norm(x, w)
    assert y.device == x.device
    want, _ = ref.norm(x, w, 1e-5)
    assert_within(y, want, want.abs() * (ref.HALF[F16] + ref.NORM_F32) + 2.0**-25)
    lp = ops.token_logprobs(x, torch.zeros(3, dtype=torch.int64, device="cuda:1"), 2)
    assert lp[0].device == x.device
