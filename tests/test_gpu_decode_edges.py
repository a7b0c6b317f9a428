"""The decode-step operators where they can go wrong: rows shorter than a chunk and more rows than a
grid has blocks, a tensor given twice, pages that are all refused, scores far apart."""

import pytest
import torch

import decode_reference as ref
from int4gemv import capi, ops
from test_gpu_decode_ops import BF16, F16, F32, assert_within, gen, no_status_left, randn, same_bits  # noqa: F401

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
