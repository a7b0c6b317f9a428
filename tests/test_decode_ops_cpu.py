"""The decode-step operators' argument checks: refused before anything touches a GPU, through the
C ABI with addresses that are never dereferenced and through the torch binding with CPU tensors."""

import ctypes

import pytest
import torch

from int4gemv import capi, ops

FAKE = 4096  # 256-byte aligned, never dereferenced: the checks fail first


def cache(**changes):
    c = capi.PagedCache(k=FAKE, v=FAKE, weights=FAKE, num_blocks=10, block_size=16, kv_heads=2,
                        head_dim=64, dtype=capi.DTYPE_F16)
    for i, s in enumerate((16 * 2 * 64, 2 * 64, 64)):
        c.k_strides[i] = c.v_strides[i] = s
    for key, value in changes.items():
        if key == "k_strides":
            for i, s in enumerate(value):
                c.k_strides[i] = s
        else:
            setattr(c, key, value)
    return c


def refused(name, *args):
    with pytest.raises(capi.CapiError) as e:
        capi.call(name, *args)
    assert e.value.code == capi.ERR_INVALID
    return str(e.value)


def test_cache_struct_layout():
    assert ctypes.sizeof(capi.PagedCache) == capi.lib().int4gemv_paged_cache_struct_bytes()


@pytest.mark.parametrize("args,message", [
    ((FAKE, FAKE, FAKE, FAKE, FAKE, 1e-5, 7, 4, 64, None), "add_rms_norm: unsupported dtype 7"),
    ((FAKE, FAKE, FAKE, FAKE, FAKE, 1e-5, 1, 4, 0, None),
     "add_rms_norm: rows = 4, hidden = 0 are out of range"),
    ((FAKE, FAKE, FAKE, FAKE, FAKE, 1e-5, 1, -1, 64, None),
     "add_rms_norm: rows = -1, hidden = 64 are out of range"),
    ((FAKE, None, FAKE, FAKE, FAKE, 1e-5, 1, 4, 64, None), "add_rms_norm: a residual needs h"),
    ((None, FAKE, FAKE, FAKE, FAKE, 1e-5, 1, 4, 64, None),
     "add_rms_norm: null pointer for a non-empty tensor"),
    ((FAKE, FAKE, FAKE + 1, FAKE, FAKE, 1e-5, 1, 4, 64, None),
     "add_rms_norm: x, residual, weight and h must be aligned to an element"),
])
def test_norm_argument_errors(args, message):
    assert refused("int4gemv_add_rms_norm", *args) == message


def test_norm_empty():
    assert capi.lib().int4gemv_add_rms_norm(None, None, None, None, None, 1e-5, 1, 0, 64, None) == 0
    assert refused("int4gemv_add_rms_norm_quant", FAKE, None, None, FAKE, None, FAKE, 1e-5, 1, 4, 64,
                   None) == "add_rms_norm_quant: null pointer for a non-empty tensor"


def attend(c, batch=3, q_heads=4, max_blocks=5, q=FAKE, k_new=None, v_new=None, ws=FAKE,
           ws_bytes=1 << 40):
    return refused("int4gemv_paged_attention", FAKE, q, ctypes.addressof(c), FAKE, FAKE, 1.0, k_new,
                   v_new, 1, batch, q_heads, max_blocks, ws, ws_bytes, None)


@pytest.mark.parametrize("changes,message", [
    (dict(head_dim=60), "head_dim 60 must be a multiple of 8 in [8, 256]"),
    (dict(head_dim=264), "head_dim 264 must be a multiple of 8 in [8, 256]"),
    (dict(dtype=0), "unsupported dtype 0"),
    (dict(block_size=0), "num_blocks = 10, block_size = 0, kv_heads = 2 are out of range"),
    (dict(k=FAKE + 8), "k and v must be 16-byte aligned, weights 4-byte"),
    (dict(k_strides=(2052, 128, 64)), "the caches' strides must be non-negative multiples of 8 elements"),
    (dict(k_strides=(2048, -128, 64)), "the caches' strides must be non-negative multiples of 8 elements"),
    (dict(k=None), "null pointer for a non-empty tensor"),
    (dict(weights=None), "null pointer for a non-empty tensor"),
])
def test_cache_argument_errors(changes, message):
    assert attend(cache(**changes)) == "paged_attention: " + message
    c = cache(**changes)
    assert refused("int4gemv_paged_evict", FAKE, FAKE, ctypes.addressof(c), FAKE, FAKE, FAKE, 16, 4,
                   3, 5, 1, None) == "paged_evict: " + message


def test_attention_argument_errors():
    c = cache()
    assert attend(c, q_heads=5) == "paged_attention: q_heads 5 must be a multiple of kv_heads 2"
    assert "batch = 70000" in attend(c, batch=70000)
    assert "out of range" in attend(c, max_blocks=2**30)
    assert attend(c, k_new=FAKE) == "paged_attention: k_new and v_new come together"
    assert attend(c, q=FAKE + 4) == ("paged_attention: q, out, k_new and v_new must be 16-byte aligned")
    size = capi.lib().int4gemv_paged_attention_workspace_size
    need = size(ctypes.addressof(c), 3, 4, 5, 1)
    assert need > size(ctypes.addressof(c), 3, 4, 5, 0) >= 0
    for ws, have in ((None, need), (FAKE, need - 1), (FAKE + 16, need)):
        with pytest.raises(capi.CapiError, match=f"workspace of {need} bytes") as e:
            capi.call("int4gemv_paged_attention", FAKE, FAKE, ctypes.addressof(c), FAKE, FAKE, 1.0,
                      None, None, 1, 3, 4, 5, ws, have, None)
        assert e.value.code == capi.ERR_WORKSPACE
    assert size(ctypes.addressof(cache(head_dim=12)), 3, 4, 5, 0) == -1
    assert size(ctypes.addressof(c), 0, 4, 5, 0) == 0
    assert capi.lib().int4gemv_paged_attention(None, None, ctypes.addressof(c), None, None, 1.0, None,
                                               None, 0, 0, 4, 5, None, 0, None) == capi.OK


@pytest.mark.parametrize("budget,recent,blocks,message", [
    (0, 0, 1, "budget 0 must be positive and recent 0 in [0, budget]"),
    (8, 9, 1, "budget 8 must be positive and recent 9 in [0, budget]"),
    (8, -1, 1, "budget 8 must be positive and recent -1 in [0, budget]"),
    (17, 4, 1, "the new table has room for 16 positions, the budget is 17"),
])
def test_evict_argument_errors(budget, recent, blocks, message):
    c = cache()
    assert refused("int4gemv_paged_evict", FAKE, FAKE, ctypes.addressof(c), FAKE, FAKE, FAKE, budget,
                   recent, 3, 5, blocks, None) == "paged_evict: " + message


@pytest.mark.parametrize("dtype,rows,vocab,stride,top,message", [
    (5, 1, 100, 100, 0, "unsupported dtype 5"),
    (1, 1, 0, 0, 0, "rows = 1, vocab = 0, row_stride = 0 are out of range"),
    (1, 1, 100, 100, 33, "top 33 must be in [0, 32] and at most vocab = 100"),
    (1, 1, 4, 4, 5, "top 5 must be in [0, 32] and at most vocab = 4"),
    (1, 1, 4, 4, -1, "top -1 must be in [0, 32] and at most vocab = 4"),
])
def test_logprobs_argument_errors(dtype, rows, vocab, stride, top, message):
    assert refused("int4gemv_token_logprobs", FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, dtype, rows, vocab,
                   stride, top, None) == "token_logprobs: " + message
    assert refused("int4gemv_token_logprobs", FAKE, FAKE, None, FAKE, FAKE, FAKE, 1, 1, 100, 100, 3,
                   None) == "token_logprobs: null pointer for a non-empty tensor"


def test_torch_binding_refuses_cpu_tensors():
    h = torch.zeros(2, 64, dtype=torch.float16)
    kv = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    ints = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros(2, 3, dtype=torch.int32)
    weights = torch.zeros(4, 2, 16)
    for call in (lambda: ops.add_rms_norm(h, h[0]), lambda: ops.add_rms_norm_quant(h, h[0]),
                 lambda: ops.paged_attention(kv[0, :2].repeat(1, 2, 1), kv, kv, table, ints, 1.0),
                 lambda: ops.paged_evict(kv, kv, weights, table, ints, table, 8, 2),
                 lambda: ops.token_logprobs(h, torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_torch_binding_signatures():
    for name, args in (("add_rms_norm", ("x", "weight", "eps", "residual")),
                       ("paged_attention", ("q", "k_cache", "v_cache", "block_table", "seq_lens",
                                            "scale", "k", "v", "weights")),
                       ("paged_evict", ("k_cache", "v_cache", "weights", "block_table", "seq_lens",
                                        "new_table", "budget", "recent")),
                       ("token_logprobs", ("logits", "tokens", "top"))):
        doc = getattr(ops, name).__doc__
        assert all(f"{a}:" in doc for a in args), doc
