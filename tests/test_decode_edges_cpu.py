"""Calls of the decode-step operators at the limits of their arguments, refused on the host."""

import ctypes

import pytest

from int4gemv import capi

from test_decode_ops_cpu import FAKE, cache, refused


@pytest.mark.parametrize("block_size,max_blocks,new_blocks,budget", [
    (2**31 - 1, 1, 1, 2**31 - 1),  # outputs: the loop over a row of `kept` stepped past 2^31
    (2**31 - 1, 0, 1, 2**31 - 500),
    (1, 2**31 - 1, 16, 16),  # lengths: so did the loops over a sequence's positions
    (2**31 - 8191, 1, 1, 16),
])
def test_evict_refuses_positions_near_the_end_of_32_bits(block_size, max_blocks, new_blocks, budget):
    c = cache(block_size=block_size, kv_heads=1)
    message = refused("int4gemv_paged_evict", FAKE, FAKE, ctypes.addressof(c), FAKE, FAKE, FAKE, budget, 4,
                      1, max_blocks, new_blocks, None)
    assert message.startswith("paged_evict: batch = 1 with tables of") and message.endswith("out of range")


def test_the_same_tensor_twice_is_refused():
    """Outputs in the place of tensors that other blocks still read."""
    other = FAKE * 2
    for y, h, x, residual in ((FAKE, FAKE, other, other), (other, other, other, None)):
        assert refused("int4gemv_add_rms_norm", y, h, x, residual, FAKE * 3, 1e-5, 1, 4, 64, None) == (
            "add_rms_norm: y must not be h, nor x or residual where it is of 8 bits")
    for y, x, residual in ((FAKE, FAKE, other), (FAKE, other, FAKE)):
        assert refused("int4gemv_add_rms_norm_quant", y, FAKE * 3, FAKE * 4, x, residual, FAKE * 5, 1e-5, 1,
                       4, 64, None) == (
            "add_rms_norm_quant: y must not be h, nor x or residual where it is of 8 bits")
    c = cache()
    assert refused("int4gemv_paged_attention", FAKE, FAKE, ctypes.addressof(c), FAKE, FAKE, 1.0, None, None,
                   0, 3, 4, 5, FAKE, 1 << 40, None) == "paged_attention: out must not be q"
    for lens, new_table in ((other, FAKE * 4), (FAKE * 5, FAKE * 3)):
        assert refused("int4gemv_paged_evict", FAKE, other, ctypes.addressof(c), FAKE * 3, lens,
                       new_table, 16, 4, 3, 5, 1, None) == (
            "paged_evict: new_lens must not be seq_lens, nor new_table block_table")


@pytest.mark.parametrize("head_dim,group,counted", [(64, 4, 4), (128, 5, 6), (128, 16, 16), (64, 17, 32), (256, 3, 4),
                                                    (192, 9, 16)])
def test_workspace_of_weights_is_what_the_header_says(head_dim, group, counted):
    """4 bytes a sequence, position of the table and counted query head, beside what a call without takes."""
    size = capi.lib().int4gemv_paged_attention_workspace_size
    for batch, blocks in ((3, 24), (40, 240)):  # 384 and 3840 positions, whole tiles of any kernel
        a = ctypes.addressof(c := cache(head_dim=head_dim))
        plain = size(a, batch, 2 * group, blocks, 0)
        scores = 4 * batch * c.kv_heads * blocks * 16 * counted
        assert 0 <= plain < 6 << 20
        assert scores <= size(a, batch, 2 * group, blocks, 1) < scores + (6 << 20)
